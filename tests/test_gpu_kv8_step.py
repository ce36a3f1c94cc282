"""Steps of a server with an 8-bit cache, its operators in the order they run: append a prompt
(heads normed and rotated), attend, project and sample; then a drafted tree behind it, then the
accepted tokens over the tree's slots. Each stage against 64 bits from what the stage before
left on the device; and the drafted step captured and replayed."""
import math

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import ops
from tests import kv8_ref, serving_ref as ref
from tests.helpers import bits_equal, gen, randn
from tests.test_gpu_kv8_attention import on_tensor_cores

pytestmark = pytest.mark.gpu

HQ, HKV, HD, PAGE, BLOCK, VOCAB, THETA, SEQS = 8, 2, 64, 32, 16, 2000, 5e5, 3


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Server:
    def __init__(self, cuda, dtype, interleaved):
        g = gen(1)
        self.cuda, self.dtype, self.interleaved = cuda, dtype, interleaved
        model = kv8_ref.Cache(SEQS * 8 + 1, HKV, PAGE, HD, BLOCK)
        self.ids = torch.randperm(SEQS * 8 + 1, generator=g)[:SEQS * 8].view(SEQS, 8).to(torch.int32)
        self.cache = ops.PagedKV8(*model.tensors(cuda), self.ids.to(cuda))
        self.table = ops.RopeTable(256, HD, THETA, cuda, scaling=ops.RopeScaling("linear", 2.0))
        self.wq, self.wk = (randn((HD,), dtype, g, scale=0.3, offset=1.0) for _ in range(2))
        self.w = randn((HQ * HD, VOCAB), dtype, g, scale=0.2)
        self.dq, self.dk, self.dw = self.wq.to(cuda), self.wk.to(cuda), self.w.to(cuda)
        self.status = ops.DeviceStatus(cuda)
        self.g = g

    def step(self, qkv, ctx, starts, most_ctx, most, positions, mask, uniforms):
        """The calls of one step."""
        q = ops.paged_kv8_append(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], self.cache, ctx, starts, most,
                                 positions=positions, table=self.table, q_weight=self.dq, k_weight=self.dk,
                                 interleaved=self.interleaved, status=self.status)
        out = ops.paged_kv8_tree_attention(q, self.cache, ctx, starts, most_ctx, most, tree_mask=mask, status=self.status)
        logits = ops.gemm(out.view(-1, HQ * HD), self.dw)
        return q, out, logits, ops.sample(logits, uniforms, status=self.status)

    def values(self):
        out = []
        for codes, scales in ((self.cache.k_pages, self.cache.k_scales), (self.cache.v_pages, self.cache.v_scales)):
            e = np.clip(scales.view(torch.uint8).cpu().numpy().astype(np.int64) - 127, -40, 40)
            v = kv8_ref.VALUES[codes.view(torch.uint8).cpu().numpy()] * np.repeat(2.0 ** e, BLOCK, axis=2)[..., None]
            out.append((v, e))
        return out

    def check(self, qkv, ctx, starts, positions, mask, uniforms, got):
        q, out, logits, tokens = got
        assert self.status.read() == 0
        freq = ref.frequencies(HD, THETA, "linear", 2.0)
        turn = lambda x, w: kv8_ref.turned(x, w, 1e-5, positions, freq, self.interleaved)  # noqa: E731
        want, off = turn(qkv[:, :HQ], self.wq)
        assert np.all(np.abs(q.cpu().double().numpy() - want) <= off + ref.HALF[self.dtype] * (np.abs(want) + off) * 1.01)
        (k, ke), (v, ve) = self.values()
        wk, koff = turn(qkv[:, HQ:HQ + HKV], self.wk)
        wv = qkv[:, HQ + HKV:].double().numpy()
        for b, c in enumerate(ctx):
            for i in range(starts[b + 1] - starts[b]):
                p, o, r = int(self.ids[b, (c + i) // PAGE]), (c + i) % PAGE, starts[b] + i
                for got_, e, x, dx in ((k, ke, wk[r], koff[r]), (v, ve, wv[r], np.zeros_like(wv[r]))):
                    step = kv8_ref.half_step(np.abs(x) + dx, e[p, :, o // BLOCK][:, None])
                    assert np.all(np.abs(got_[p, :, o] - x) <= step + dx)
        seen = (lambda row, i, j: j <= i) if mask is None else (lambda row, i, j: bool((int(mask[row, 0]) >> j) & 1))
        k, v = (torch.from_numpy(np.nan_to_num(x)) for x in (k, v))
        tc = on_tensor_cores(self.dtype, HD, PAGE, BLOCK)
        want, tol = ref.attention(q, k, v, self.ids, list(range(SEQS)), ctx, starts, seen, 1 / math.sqrt(HD), self.dtype, tc)
        if tc:  # the parts of queries and weights: 2^-17 of a score's terms, 2^-11 and 2^-16 of weights
            size = q.cpu().double().abs().amax(-1, keepdim=True).numpy() * HD * float(k.abs().max()) / math.sqrt(HD)
            tol = tol + (2 * 2.0 ** -17 * size + 2.0 ** -11 + 2.0 ** -16 * (max(ctx) + max(np.diff(starts)))) * float(v.abs().max())
        assert np.all(np.abs(out.cpu().double().numpy() - want) <= tol)
        o, w = out.cpu().double().view(len(qkv), -1).numpy(), self.w.double().numpy()
        # fp32 accumulation of HQ * HD products, rounded once to the type
        bound = (HQ * HD) * 2.0 ** -24 * (np.abs(o) @ np.abs(w)) + 1.01 * ref.HALF[self.dtype] * np.abs(o @ w)
        assert np.all(np.abs(logits.cpu().double().numpy() - o @ w) <= bound)
        assert tokens.cpu().tolist() == ref.sample(logits, uniforms, None, None, None, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_steps_stage_by_stage(cuda, dtype, interleaved):
    s = Server(cuda, dtype, interleaved)
    # prompts of uneven lengths, a drafted tree behind each, then the accepted tokens and one more
    prompts = [37, 130, 5]
    parents = [[-1, 0, 0, 1], [-1, -1, 1, 2, 0, 4], []]
    depth = []
    for p in parents:
        d = []
        for j in p:
            d.append(d[j] + 1 if j >= 0 else 0)
        depth.append(d)
    bits = torch.cat([ref.tree_bits(p, 1) for p in parents if p])
    plain = [([0, 0, 0], prompts, None, None), (prompts, [len(p) for p in parents], depth, bits), (prompts, [3, 4, 1], None, None)]
    for ctx, counts, d, mask in plain:
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        rows = starts[-1]
        qkv = randn((rows, HQ + 2 * HKV, HD), dtype, s.g, scale=2.0)
        positions = [c + (d[b][i] if d else i) for b, c in enumerate(ctx) for i in range(counts[b])]
        u = torch.rand(rows, generator=s.g)
        got = s.step(qkv.to(cuda), i32(ctx, cuda), i32(starts, cuda), max(ctx), max(counts), i32(positions, cuda) if d else None,
                     None if mask is None else mask.to(cuda), u.to(cuda))
        s.check(qkv, ctx, starts, positions, mask, u, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_captured_step(cuda, dtype):
    """The step in a graph gives what the calls give, on the inputs and lengths of its replay."""
    s = Server(cuda, dtype, False)
    prompts, starts0 = [40, 64, 17], [0, 40, 104, 121]
    s.step(randn((121, HQ + 2 * HKV, HD), dtype, s.g).to(cuda), i32([0, 0, 0], cuda), i32(starts0, cuda), 0, 64, None, None,
           torch.rand(121, generator=s.g).to(cuda))
    qkv = randn((SEQS, HQ + 2 * HKV, HD), dtype, s.g).to(cuda)
    ctx, starts, u = i32(prompts, cuda), i32([0, 1, 2, 3], cuda), torch.rand(SEQS, generator=s.g).to(cuda)
    names = ("k_pages", "v_pages", "k_scales", "v_scales")
    keep = [getattr(s.cache, n).view(torch.uint8).clone() for n in names]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = s.step(qkv, ctx, starts, 200, 1, None, None, u)
    for turn in range(3):
        for n, t in zip(names, keep):
            getattr(s.cache, n).view(torch.uint8).copy_(t)
        want = [t.clone() for t in s.step(qkv, ctx, starts, 200, 1, None, None, u)]
        after = [getattr(s.cache, n).view(torch.uint8).clone() for n in names]
        for n, t in zip(names, keep):
            getattr(s.cache, n).view(torch.uint8).copy_(t)
        graph.replay()
        assert all(bits_equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(getattr(s.cache, n).view(torch.uint8), t) for n, t in zip(names, after))
        keep = after
        ctx.add_(1)
        qkv.copy_(randn((SEQS, HQ + 2 * HKV, HD), dtype, s.g))
    assert s.status.read() == 0


def test_the_cache_read_back_into_a_16_bit_one(cuda):
    """A prefix taken out of an 8-bit cache, appended to a bf16 one: attention over either gives the
    same values up to its own roundings."""
    s = Server(cuda, torch.bfloat16, False)
    starts = [0, 50, 130, 137]
    qkv = randn((137, HQ + 2 * HKV, HD), torch.bfloat16, s.g).to(cuda)
    s.step(qkv, i32([0, 0, 0], cuda), i32(starts, cuda), 0, 80, None, None, torch.rand(137, generator=s.g).to(cuda))
    k, v = ops.paged_kv8_read(s.cache, i32([0, 0, 0], cuda), i32(starts, cuda), 137, 80)
    pages = [torch.zeros(SEQS * 8 + 1, HKV, PAGE, HD, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    wide = ops.PagedKV(*pages, s.cache.page_table)
    seqs = i32([b for b in range(3) for _ in range(starts[b + 1] - starts[b])], cuda)
    slots = i32([t for b in range(3) for t in range(starts[b + 1] - starts[b])], cuda)
    ops.paged_kv_append(None, k, v, None, wide, seq_ids=seqs, slots=slots)
    q = randn((3, HQ, HD), torch.bfloat16, s.g).to(cuda)
    args = (i32([49, 79, 6], cuda), i32([0, 1, 2, 3], cuda), 79, 1)
    a, b = ops.paged_kv8_tree_attention(q, s.cache, *args), ops.paged_tree_attention(q, wide, *args)
    # each off by half a step of its weights and of the output, and the parts' 2^-11 and 2^-12
    assert float((a.float() - b.float()).abs().max()) <= 5 * 2.0 ** -8 * float(v.float().abs().max())
