"""A decode step with drafted tokens, the operators in the order a server runs them: append
the tree's keys and values to the paged cache (rotating q and k), attend, project to
the vocabulary (ops.gemm), sample a token per row; then append the accepted tokens again
at their positions and go on without a mask. Each stage against 64 bits, from the inputs that
the stage before left on the device; and the whole step captured and replayed."""
import math

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import ops
from tests import serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

HQ, HKV, HD, PAGE, VOCAB, THETA = 8, 2, 64, 16, 2000, 5e5


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Step:
    def __init__(self, cuda, dtype, interleaved, seed):
        g = gen(seed)
        self.cuda, self.dtype, self.interleaved = cuda, dtype, interleaved
        self.ctx = [37, 0, 130, 5]
        self.parents = [[-1, 0, 0, 1], [-1, 0], [-1, -1, 1, 2, 0, 4], []]
        self.n = [len(p) for p in self.parents]
        self.rows = sum(self.n)
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).tolist()
        width = max(-(-(c + n + 8) // PAGE) for c, n in zip(self.ctx, self.n))
        self.ids = torch.randperm(4 * width, generator=g).view(4, width)
        # stale contents everywhere but in the contexts: NaN
        self.k, self.v = (torch.full((4 * width, HKV, PAGE, HD), math.nan, dtype=dtype) for _ in range(2))
        for b, c in enumerate(self.ctx):
            for t in range(c):
                for x in (self.k, self.v):
                    x[self.ids[b, t // PAGE], :, t % PAGE] = randn((HKV, HD), dtype, g)
        depth = []
        for p in self.parents:
            d = []
            for j in p:
                d.append(d[j] + 1 if j >= 0 else 0)
            depth.append(d)
        self.seqs = [b for b in range(4) for _ in range(self.n[b])]
        self.slots = [self.ctx[b] + j for b in range(4) for j in range(self.n[b])]
        self.pos = [self.ctx[b] + d for b in range(4) for d in depth[b]]
        self.mask = torch.cat([ref.tree_bits(p, 1) for p in self.parents if p])
        self.qkv = randn((self.rows, HQ + 2 * HKV, HD), dtype, g)
        self.w = randn((HQ * HD, VOCAB), dtype, g, scale=0.2)
        self.u = torch.rand(self.rows, generator=g)
        pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (self.rows,), generator=g)]  # noqa: E731
        self.settings = dict(temperature=pick([0.0, 0.7, 1.0]), top_k=pick([0, 1, 40]).to(torch.int32),
                             top_p=pick([0.9, 1.0]), min_p=pick([0.0, 0.05]))
        self.table = ops.RopeTable(512, HD, THETA, cuda, scaling=ops.RopeScaling("linear", 2.0))

    def device(self):
        c = self.cuda
        self.cache = ops.PagedKV(self.k.to(c), self.v.to(c), self.ids.to(torch.int32).to(c))
        self.d = dict(qkv=self.qkv.to(c), pos=i32(self.pos, c), slots=i32(self.slots, c), seqs=i32(self.seqs, c),
                      ctx=i32(self.ctx, c), starts=i32(self.starts, c), mask=self.mask.to(c), w=self.w.to(c), u=self.u.to(c),
                      **{n: t.to(c) for n, t in self.settings.items()})
        self.status = ops.DeviceStatus(c)

    def run(self):
        d = self.d
        q, k, v = d["qkv"][:, :HQ], d["qkv"][:, HQ:HQ + HKV], d["qkv"][:, HQ + HKV:]
        q = ops.paged_kv_append(q, k, v, d["pos"], self.cache, table=self.table, seq_ids=d["seqs"], slots=d["slots"],
                                interleaved=self.interleaved, status=self.status)
        out = ops.paged_tree_attention(q, self.cache, d["ctx"], d["starts"], max(self.ctx), max(self.n), tree_mask=d["mask"],
                                       status=self.status)
        logits = ops.gemm(out.view(self.rows, HQ * HD), d["w"])
        tokens = ops.sample(logits, d["u"], d["temperature"], d["top_k"], d["top_p"], d["min_p"], status=self.status)
        return q, out, logits, tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_step_stage_by_stage(cuda, dtype, interleaved):
    s = Step(cuda, dtype, interleaved, 1)
    s.device()
    q, out, logits, tokens = s.run()
    assert s.status.read() == 0
    f = ref.frequencies(HD, THETA, "linear", 2.0)
    want, pair = ref.rotated(s.qkv[:, :HQ], s.pos, f, 1.0, interleaved)
    assert np.all(np.abs(q.cpu().double().numpy() - want) <= ref.rotation_tolerance(want, pair, 1.0, dtype))
    wk, pair = ref.rotated(s.qkv[:, HQ:HQ + HKV], s.pos, f, 1.0, interleaved)
    kc, vc = s.cache.k_pages.cpu(), s.cache.v_pages.cpu()
    for r, (b, t) in enumerate(zip(s.seqs, s.slots)):
        got = kc[s.ids[b, t // PAGE], :, t % PAGE].double().numpy()
        assert np.all(np.abs(got - wk[r]) <= ref.rotation_tolerance(wk[r], pair[r], 1.0, dtype))
        assert bits_equal(vc[s.ids[b, t // PAGE], :, t % PAGE], s.qkv[r, HQ + HKV:])
    bits = s.mask.numpy()
    want, tol = ref.attention(q, kc, vc, s.ids, list(range(4)), s.ctx, s.starts,
                              lambda row, i, j: bool((int(bits[row, 0]) >> j) & 1), 1 / math.sqrt(HD), dtype,
                              dtype == torch.bfloat16)
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= tol)
    o, w = out.cpu().double().view(s.rows, -1).numpy(), s.w.double().numpy()
    # fp32 accumulation of HQ * HD products, rounded once to the type
    bound = (HQ * HD) * 2.0 ** -24 * (np.abs(o) @ np.abs(w)) + 1.01 * ref.HALF[dtype] * np.abs(o @ w)
    assert np.all(np.abs(logits.cpu().double().numpy() - o @ w) <= bound)
    assert tokens.cpu().tolist() == ref.sample(logits, s.u, **s.settings)

    # Sequence 2 accepts nodes 1, 2 and 3 (slots 1, 2, 3 of the tree, positions 130..132):
    # their keys and values go to the slots of their positions, and a new token attends.
    rows = [s.starts[2] + j for j in (1, 2, 3)]
    d = s.d["qkv"][rows]
    ops.paged_kv_append(None, d[:, HQ:HQ + HKV], d[:, HQ + HKV:], i32([130, 131, 132], cuda), s.cache, table=s.table,
                        seq_ids=i32([2, 2, 2], cuda), interleaved=interleaved, status=s.status)
    new = randn((1, HQ + 2 * HKV, HD), dtype, gen(9)).to(cuda)
    q = ops.paged_kv_append(new[:, :HQ], new[:, HQ:HQ + HKV], new[:, HQ + HKV:], i32([133], cuda), s.cache, table=s.table,
                            seq_ids=i32([2], cuda), interleaved=interleaved, status=s.status)
    out = ops.paged_tree_attention(q, s.cache, i32([133], cuda), i32([0, 1], cuda), 133, 1, seq_ids=i32([2], cuda),
                                   status=s.status)
    assert s.status.read() == 0
    want, tol = ref.attention(q, s.cache.k_pages, s.cache.v_pages, s.ids, [2], [133], [0, 1], lambda *_: True,
                              1 / math.sqrt(HD), dtype, dtype == torch.bfloat16)
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_step_replays_with_new_inputs(cuda, dtype):
    s, t = Step(cuda, dtype, False, 2), Step(cuda, dtype, False, 3)
    t.device()
    want = [x.clone() for x in t.run()]
    s.device()
    s.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run()
    for n, x in t.d.items():
        s.d[n].copy_(x)
    s.cache.k_pages.copy_(t.k.to(cuda))
    s.cache.v_pages.copy_(t.v.to(cuda))
    s.cache.page_table.copy_(t.ids.to(torch.int32).to(cuda))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert bits_equal(a, b)
    assert s.status.read() == 0


def test_two_steps_at_once_on_their_own_streams(cuda):
    """Two batches' steps on two streams: each has its own cache and scratch."""
    steps = [Step(cuda, torch.bfloat16, False, 4), Step(cuda, torch.bfloat16, True, 5)]
    want = []
    for s in steps:
        s.device()
        want.append([x.clone() for x in s.run()])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        got = []
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                got.append(s.run())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert bits_equal(a, b)
