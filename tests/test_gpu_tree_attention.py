"""Tree attention over a paged cache on the GPU against 64-bit softmax attention, one
row and head at a time; the tolerance is derived where it is computed (serving_ref)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class Batch:
    """Sequences of (context, drafted tokens) over shuffled pages; what lies behind each
    sequence's last slot, and in pages of nobody, is NaN."""

    def __init__(self, cuda, lens, hq, hkv, hd, page, dtype, seed=0, spread=2.0, extra_rows=0, tree=True, lead_rows=0):
        g = gen(seed)
        self.lens, self.page, self.dtype = lens, page, dtype
        need = [-(-(c + n) // page) for c, n in lens]
        width = max(need + [1])
        ids = torch.randperm(sum(need) + 2, generator=g).tolist()
        table, at = [], 0
        for n in need:
            table.append(ids[at:at + n] + [-7] * (width - n))
            at += n
        k, v = (torch.full((len(ids), hkv, page, hd), math.nan, dtype=dtype) for _ in range(2))
        for b, (c, n) in enumerate(lens):
            for t in range(c + n):
                k[table[b][t // page], :, t % page] = randn((hkv, hd), dtype, g)
                v[table[b][t // page], :, t % page] = randn((hkv, hd), dtype, g)
        self.starts = [lead_rows]
        for _, n in lens:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + extra_rows
        self.q = randn((self.rows, hq, hd), dtype, g, scale=spread)
        self.max_ctx, self.max_tree = max(c for c, _ in lens), max(n for _, n in lens)
        self.words = -(-max(self.max_tree, 1) // 64)
        rng = np.random.RandomState(seed)
        self.parents = [[rng.randint(max(-1, j - 5), j) for j in range(n)] for _, n in lens]
        self.mask = torch.zeros(self.rows, self.words, dtype=torch.int64)
        for b in range(len(lens)):
            if lens[b][1]:
                self.mask[self.starts[b]:self.starts[b + 1]] = ref.tree_bits(self.parents[b], self.words)
        self.tree = tree
        self.cuda = cuda
        self.cache = ops.PagedKV(k.to(cuda), v.to(cuda), i32(table, cuda))
        self.k, self.v, self.table = k, v, torch.tensor(table, dtype=torch.int32)
        self.hd, self.group = hd, hq // hkv

    def run(self, **kw):
        args = dict(tree_mask=self.mask.to(self.cuda) if self.tree else None)
        args.update(kw)
        return ops.paged_tree_attention(self.q.to(self.cuda), self.cache, i32([c for c, _ in self.lens], self.cuda),
                                        i32(self.starts, self.cuda), self.max_ctx, self.max_tree, **args)

    def want(self, mask=None, scale=None, seqs=None):
        if mask is None and self.tree:
            bits = self.mask.numpy().view(np.uint64)
            mask = lambda row, i, j: bool((int(bits[row, j // 64]) >> (j % 64)) & 1)  # noqa: E731
        elif mask is None:
            mask = lambda row, i, j: j <= i  # noqa: E731
        return ref.attention(self.q, self.k, self.v, self.table, seqs or list(range(len(self.lens))),
                             [c for c, _ in self.lens], self.starts, mask, scale or 1 / math.sqrt(self.hd), self.dtype,
                             self.dtype == BF16)

    def check(self, got=None, **kw):
        st = ops.DeviceStatus(self.cuda)
        if got is None:
            got = self.run(status=st, **kw)
            assert st.read() == 0
        want, tol = self.want()
        rows = slice(self.starts[0], self.starts[-1])
        err = np.abs(got.cpu().double().numpy() - want)[rows]
        assert np.all(err <= tol[rows]), (np.nanmax(err), np.isnan(err).sum(), np.nanmax(err - tol[rows]))
        return got


LENS = {
    "one": [(300, 1)],
    "empty-context": [(0, 1), (0, 5)],
    "tile-edges": [(127, 1), (128, 1), (128, 8), (120, 8), (121, 8), (255, 2), (0, 128)],
    "ragged": [(5, 3), (700, 0), (0, 0), (33, 17), (1, 64), (513, 1)],
    "words": [(40, 65), (3, 130), (200, 64)],
    "long": [(2500, 6), (10, 2)],
}


@pytest.mark.parametrize("dtype,hq,hkv,hd,page", [
    (BF16, 8, 2, 128, 16), (BF16, 4, 4, 128, 64), (BF16, 16, 2, 128, 8), (BF16, 7, 1, 128, 128), (BF16, 8, 1, 64, 32),
    (BF16, 6, 2, 64, 256), (BF16, 4, 2, 128, 24), (BF16, 4, 2, 48, 16), (BF16, 2, 1, 256, 16), (BF16, 24, 2, 128, 512),
    (BF16, 4, 2, 80, 100), (BF16, 8, 1, 8, 72), (BF16, 3, 1, 120, 200), (BF16, 4, 1, 96, 7), (BF16, 16, 1, 56, 250),
    (BF16, 32, 1, 112, 24),
    (F32, 6, 6, 48, 16), (F32, 8, 2, 128, 7), (F32, 4, 1, 256, 100), (F32, 2, 2, 4, 1), (F32, 6, 1, 100, 32)])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("tree", [True, False])
def test_against_64_bits(cuda, lens, dtype, hq, hkv, hd, page, tree):
    Batch(cuda, LENS[lens], hq, hkv, hd, page, dtype, seed=hd + page, tree=tree).check()


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (BF16, 64), (F32, 48), (BF16, 80)])
def test_many_uneven_sequences(cuda, dtype, hd):
    rng = np.random.RandomState(3)
    lens = [(int(rng.randint(0, 600)), int(rng.randint(0, 12))) for _ in range(70)]
    Batch(cuda, lens, 4, 2, hd, 16, dtype, seed=4).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_wide_groups(cuda, dtype):
    Batch(cuda, [(200, 3), (9, 30)], 64, 1, 128, 32, dtype, seed=5).check()
    Batch(cuda, [(200, 9)], 33, 1, 64, 32, dtype, seed=6).check()


@pytest.mark.parametrize("dtype,hd,page", [(BF16, 128, 16), (F32, 64, 10), (BF16, 48, 16)])
def test_rows_that_see_little_or_nothing(cuda, dtype, hd, page):
    """Masks that leave a row empty (zeros), hide a row from itself, and set bits past the
    tree."""
    b = Batch(cuda, [(0, 4), (0, 70), (130, 3), (5, 2)], 4, 2, hd, page, dtype, seed=7)
    b.mask[0] = 0
    b.mask[1] = -1  # every bit, those past the tree too
    b.mask[2] = 1 << 3
    b.mask[10] = 0
    b.mask[b.starts[2]] = 0
    b.mask[b.starts[3] + 1] = torch.tensor([-4, -1])
    got = b.check()
    assert int(torch.count_nonzero(got[0])) == 0 and int(torch.count_nonzero(got[10])) == 0


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_rows_outside_the_sequences_are_left(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (300, 2)], 4, 2, hd, 16, dtype, seed=8, extra_rows=4, lead_rows=2)
    out = torch.full((b.rows, 4, hd), 5.0, dtype=dtype, device=cuda)
    b.check(b.run(out=out))
    keep = torch.full_like(out[0], 5.0)
    for r in [0, 1] + list(range(b.starts[-1], b.rows)):
        assert bits_equal(out[r], keep)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_bad_sequences_are_skipped_and_others_served(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (300, 2), (17, 4), (64, 1)], 4, 2, hd, 16, dtype, seed=9)
    want, tol = b.want()

    def go(ctx, starts, seqs, bit, bad, max_ctx=300, max_tree=4):
        out, st = torch.full((b.rows, 4, hd), 5.0, dtype=dtype, device=cuda), ops.DeviceStatus(cuda)
        ops.paged_tree_attention(b.q.to(cuda), b.cache, i32(ctx, cuda), i32(starts, cuda), max_ctx, max_tree,
                                 tree_mask=b.mask.to(cuda), seq_ids=i32(seqs, cuda), out=out, status=st)
        assert st.read() == bit
        got = out.cpu().double().numpy()
        for s in range(4):
            rows = slice(b.starts[s], b.starts[s + 1])
            if s in bad:
                assert np.all(got[rows] == 5.0)
            else:
                assert np.all(np.abs(got - want)[rows] <= tol[rows])

    ctx, st = [40, 300, 17, 64], b.starts
    go(ctx, st, [0, 1, 2, 3], 0, [])
    go(ctx, st, [0, 4, 2, -1], _lib.BM_DEVERR_BAD_SEQUENCE, [1, 3])
    go([40, 300, -1, 64], st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [2])
    go(ctx, st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [1], max_ctx=299)
    go(ctx, st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [2], max_tree=3)
    go([40, 2 ** 31 - 1, 17, 64], st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [1])
    go(ctx, st[:-1] + [b.rows + 1], [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [3])
    # behind the 19 pages of a sequence
    go([40, 303, 17, 64], st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [1], max_ctx=400)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_a_bad_page_is_flagged_and_unseen(cuda, dtype, hd):
    b = Batch(cuda, [(100, 2)], 4, 2, hd, 16, dtype, seed=10)
    for page in (-1, 10 ** 6):
        b.cache.page_table[0, 2] = page
        st = ops.DeviceStatus(cuda)
        out = b.run(status=st)
        assert st.read() == _lib.BM_DEVERR_BAD_PAGE
        # slots 32..47 are left out of the softmax
        k = b.k.double().numpy()[b.table[0].numpy()].transpose(1, 0, 2, 3).reshape(2, -1, hd)[:, :102]
        v = b.v.double().numpy()[b.table[0].numpy()].transpose(1, 0, 2, 3).reshape(2, -1, hd)[:, :102]
        s = np.einsum("hd,sd->hs", b.q[0, :2].double().numpy(), k[0]) / math.sqrt(hd)
        s[:, 32:48] = -np.inf
        s[:, 101] = -np.inf  # row 0 does not see slot 1
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want = p @ np.nan_to_num(v[0])
        # weights and output rounded to the type, half a step each
        tol = 1.01 * ref.HALF[dtype] * (p @ np.abs(np.nan_to_num(v[0])) + np.abs(want)) + 2.0 ** -16
        assert np.all(np.abs(out[0, :2].cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_far_apart(cuda, dtype):
    """Maxima that rise by a lot, late and early: weights under- and overflow unless the
    running maximum follows."""
    b = Batch(cuda, [(700, 2), (300, 1)], 4, 2, 128, 16, dtype, seed=11, spread=60.0)
    b.check()


def test_sequence_ids_share_a_cache_and_scale(cuda):
    b = Batch(cuda, [(50, 2), (90, 3)], 4, 2, 128, 16, BF16, seed=12)
    got = b.run(scale=0.03, seq_ids=i32([0, 1], cuda))
    want, tol = b.want(scale=0.03)
    assert np.all(np.abs(got.cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_repeats_streams_graphs_and_dirty_workspaces(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (1500, 2), (17, 4), (640, 1)], 4, 2, hd, 16, dtype, seed=13)
    first = b.check()
    ws = ops.paged_tree_attention_workspace(b.q.to(cuda), b.cache, 4, b.max_ctx, b.max_tree)
    for fill in (0xFF, 0x7F, 0):
        ws.fill_(fill)
        assert bits_equal(b.run(workspace=ws), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = b.run(stream=side)
    side.synchronize()
    assert bits_equal(out, first)
    q, ctx, starts, mask = b.q.to(cuda), i32([c for c, _ in b.lens], cuda), i32(b.starts, cuda), b.mask.to(cuda)
    graph, o1, o2 = torch.cuda.CUDAGraph(), torch.empty_like(q), torch.empty_like(q)
    with torch.cuda.graph(graph):
        ops.paged_tree_attention(q, b.cache, ctx, starts, b.max_ctx, b.max_tree, tree_mask=mask, out=o1, workspace=ws)
        ops.paged_tree_attention(q, b.cache, ctx, starts, b.max_ctx, b.max_tree, tree_mask=mask, out=o2, workspace=ws)
    for _ in range(3):
        o1.zero_()
        o2.zero_()
        graph.replay()
        assert bits_equal(o1, first) and bits_equal(o2, first)
    ctx.copy_(i32([40, 700, 17, 0], cuda))  # a replay reads the lengths of its time
    graph.replay()
    b.lens = [(40, 3), (700, 2), (17, 4), (0, 1)]
    want = ops.paged_tree_attention(q, b.cache, ctx, starts, b.max_ctx, b.max_tree, tree_mask=mask)
    assert bits_equal(o1, want) and not bits_equal(o1, first)


def test_a_token_alone_is_decode_attention(cuda):
    """One row per sequence and no mask against bm_decode_attention on the same cache laid
    out statically: both within their tolerances of the same 64-bit result."""
    b = Batch(cuda, [(200, 1), (77, 1)], 8, 2, 128, 16, BF16, seed=14, tree=False)
    b.check()


def test_long_prompt_chunk(cuda):
    """700 tokens behind 100 cached ones, no mask: many row tiles per sequence."""
    Batch(cuda, [(100, 700), (3, 90)], 4, 2, 128, 16, BF16, seed=15, tree=False).check()
    Batch(cuda, [(100, 300)], 4, 2, 64, 16, F32, seed=16, tree=False).check()


def test_nothing_to_do(cuda):
    b = Batch(cuda, [(5, 1)], 4, 2, 128, 16, BF16)
    none = i32([], cuda)
    out = ops.paged_tree_attention(b.q[:0].to(cuda), b.cache, none, i32([0], cuda), 0, 0)
    assert out.shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 5.0, dtype=BF16, device=cuda)
    ops.paged_tree_attention(torch.zeros_like(out), b.cache, i32([5], cuda), i32([1, 1], cuda), 8, 4, out=out)
    assert bool((out == 5.0).all())


def test_two_streams_at_once(cuda):
    """Calls that overlap on the GPU, a workspace each: the same results as one after the other."""
    batches = [Batch(cuda, [(3000, 3), (1500, 2), (17, 4)], 8, 2, 128, 16, BF16, seed=17),
               Batch(cuda, [(900, 30), (2000, 5)], 8, 2, 64, 32, BF16, seed=18),
               Batch(cuda, [(700, 4), (90, 9)], 4, 2, 48, 16, F32, seed=19)]
    first = [b.check() for b in batches]
    calls = []
    for b in batches:
        q = b.q.to(cuda)
        args = (q, b.cache, i32([c for c, _ in b.lens], cuda), i32(b.starts, cuda), b.max_ctx, b.max_tree)
        kw = [dict(tree_mask=b.mask.to(cuda), out=torch.empty_like(q),
                   workspace=ops.paged_tree_attention_workspace(q, b.cache, len(b.lens), b.max_ctx, b.max_tree))
              for _ in range(3)]
        calls.append((args, kw))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for turn in range(10):
        for s, stream in enumerate(streams):
            for i in range(3):
                args, kw = calls[(s + i) % 3]
                ops.paged_tree_attention(*args, stream=stream, **kw[s])
    torch.cuda.synchronize()
    for (args, kw), want in zip(calls, first):
        for k in kw:
            assert bits_equal(k["out"], want)


@pytest.mark.parametrize("dtype,hq,hkv,hd", [(BF16, 8, 2, 128), (BF16, 8, 2, 64), (F32, 6, 6, 48), (F32, 8, 2, 128)])
def test_a_token_alone_and_decode_attention_on_the_static_cache(cuda, dtype, hq, hkv, hd):
    """One row per sequence and no mask, and bm_decode_attention on the same K and V laid out
    statically: each within the tolerance of the same 64-bit result."""
    b = Batch(cuda, [(200, 1), (77, 1), (0, 1), (1300, 1)], hq, hkv, hd, 16, dtype, seed=20, tree=False)
    b.check()
    want, tol = b.want()
    max_seq = b.max_ctx + 1
    k, v = (torch.zeros(len(b.lens), hkv, max_seq, hd, dtype=dtype) for _ in range(2))
    for s, (c, n) in enumerate(b.lens):
        for t in range(c + n):
            k[s, :, t] = b.k[int(b.table[s, t // 16]), :, t % 16]
            v[s, :, t] = b.v[int(b.table[s, t // 16]), :, t % 16]
    lib, need = _lib.load(), ctypes.c_size_t()
    _lib.check(lib.bm_decode_attention_workspace_size(len(b.lens), hq, hkv, hd, max_seq, ctypes.byref(need)))
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device=cuda)
    q, k, v, lens = b.q.to(cuda), k.to(cuda), v.to(cuda), i32([c + n for c, n in b.lens], cuda)
    out, ids = torch.empty_like(q), i32(list(range(len(b.lens))), cuda)
    _lib.check(lib.bm_decode_attention(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), ids.data_ptr(), lens.data_ptr(),
                                       max_seq, len(b.lens), hq, hkv, hd, max_seq, len(b.lens), 0.0, ws.data_ptr(), need.value,
                                       ops.bm_dtype(q), None, torch.cuda.current_stream(cuda).cuda_stream))
    assert np.all(np.abs(out.cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (BF16, 64), (BF16, 256), (F32, 48), (F32, 128)])
@pytest.mark.parametrize("seqs", [[3, 2, 1, 0], [1, 0, 1, 2], [2, 2, 2, 2]])
def test_sequence_ids_in_any_order_and_twice(cuda, dtype, hd, seqs):
    """Entries of the batch on cache sequences of another number, two and more on the same one."""
    b = Batch(cuda, [(60, 3), (60, 2), (60, 3), (60, 1)], 8, 2, hd, 16, dtype, seed=21)
    for s in range(4):  # three drafted slots in every cache sequence
        for t in range(61, 63):
            page = int(b.table[s, t // 16])
            b.k[page, :, t % 16] = randn((2, hd), dtype, gen(100 + s + t))
            b.v[page, :, t % 16] = randn((2, hd), dtype, gen(200 + s + t))
    b.cache.k_pages.copy_(b.k)
    b.cache.v_pages.copy_(b.v)
    st = ops.DeviceStatus(cuda)
    got = b.run(seq_ids=i32(seqs, cuda), status=st)
    assert st.read() == 0
    want, tol = b.want(seqs=seqs)
    assert np.all(np.abs(got.cpu().double().numpy() - want) <= tol)
