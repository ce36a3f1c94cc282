"""The 8-bit paged cache on the GPU: what the append writes, against codes computed one block and
head at a time in 64 bits, and what the read gives back. V, and K without norm and rotation, are
quantised from the given values: their codes and scales have to be the very ones. A normed or
rotated K is off by what kv8_ref derives before it is rounded to a code."""
import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import kv8_ref, serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
THETA = 1e4


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


class State:
    """A cache that the tests fill by calls, beside its model in 64 bits."""

    def __init__(self, cuda, seqs, slots, hkv, hd, page, block, dtype, seed=0, rd=0, interleaved=False, norm=False, spare=2):
        self.cuda, self.dtype, self.hkv, self.hd, self.g = cuda, dtype, hkv, hd, gen(seed)
        width = max(1, -(-slots // page))
        self.table = torch.randperm(seqs * width + spare, generator=self.g)[:seqs * width].view(seqs, width).to(torch.int32)
        self.model = kv8_ref.Cache(seqs * width + spare, hkv, page, hd, block)
        self.cache = ops.PagedKV8(*self.model.tensors(cuda), self.table.to(cuda))
        self.rd, self.interleaved = rd, interleaved
        self.rope = ops.RopeTable(max(slots, 1), rd, THETA, cuda) if rd else None
        self.freq = ref.frequencies(rd, THETA) if rd else None
        self.wk = randn((hd,), dtype, self.g, scale=0.3, offset=1.0) if norm else None
        self.wq = randn((hd,), dtype, self.g, scale=0.3, offset=1.0) if norm else None

    def heads(self, rows, hq=0, sizes=None):
        x = randn((rows, hq + 2 * self.hkv, self.hd), self.dtype, self.g)
        if sizes is not None:
            x = (x.float() * torch.tensor(sizes)[:, None, None]).to(self.dtype)
        return x

    def append(self, x, hq, ctx, counts, seqs=None, positions=None, check=True, lead=0, **kw):
        """Rows `lead` and on of x [rows, hq + 2 hkv, hd] to the sequences, then both sides compared."""
        starts = np.concatenate([[lead], lead + np.cumsum(counts)]).tolist()
        d, st = x.to(self.cuda), ops.DeviceStatus(self.cuda)
        pos = None if positions is None else i32(positions, self.cuda)
        got = ops.paged_kv8_append(
            d[:, :hq] if hq else None, d[:, hq:hq + self.hkv], d[:, hq + self.hkv:], self.cache, i32(ctx, self.cuda),
            i32(starts, self.cuda), max(counts), positions=pos, table=self.rope,
            q_weight=self.wq.to(self.cuda) if self.wq is not None and hq else None,
            k_weight=None if self.wk is None else self.wk.to(self.cuda), eps=1e-4, interleaved=self.interleaved,
            seq_ids=None if seqs is None else i32(seqs, self.cuda), status=st, **kw)
        if not check:
            return got, st.read()
        assert st.read() == 0
        slot = np.zeros(len(x), dtype=np.int64)
        for b, c in enumerate(ctx):
            slot[starts[b]:starts[b + 1]] = c + np.arange(counts[b])
        where = slot if positions is None else np.array(positions)
        k, off = kv8_ref.turned(x[:, hq:hq + self.hkv], self.wk, 1e-4, where, self.freq, self.interleaved)
        v = x[:, hq + self.hkv:].double().numpy()
        before = [[c.copy() for c in self.model.codes], [s.copy() for s in self.model.scales]]
        unsure = np.zeros(k.shape[:2], dtype=bool)
        for b, c in enumerate(ctx):
            rows = slice(starts[b], starts[b + 1])
            pages = self.table[b if seqs is None else seqs[b]].numpy()
            unsure[rows] = self.model.append(0, pages, c, k[rows], off[rows])
            self.model.append(1, pages, c, v[rows], np.zeros_like(v[rows]))
        assert unsure.mean() < 0.01
        self.compare(k, off, ctx, starts, seqs, unsure, before)
        if hq:
            want, qoff = kv8_ref.turned(x[:, :hq], self.wq, 1e-4, where, self.freq, self.interleaved)
            tol = qoff + ref.HALF[self.dtype] * (np.abs(want) + qoff) * 1.01
            rows = slice(starts[0], starts[-1])
            assert np.all(np.abs(got.cpu().double().numpy() - want)[rows] <= tol[rows])
        return got

    def compare(self, k, off, ctx, starts, seqs, unsure, before):
        codes = [t.view(torch.uint8).cpu().numpy() for t in (self.cache.k_pages, self.cache.v_pages)]
        scales = [t.view(torch.uint8).cpu().numpy() for t in (self.cache.k_scales, self.cache.v_scales)]
        assert np.array_equal(codes[1], self.model.codes[1]) and np.array_equal(scales[1], self.model.scales[1])
        if not off.any():
            assert np.array_equal(codes[0], self.model.codes[0]) and np.array_equal(scales[0], self.model.scales[0])
            return
        page, block = self.model.page, self.model.block
        new = np.zeros(codes[0].shape[:3], dtype=bool)
        for b, c in enumerate(ctx):
            pages = self.table[b if seqs is None else seqs[b]].numpy()
            for i in range(starts[b + 1] - starts[b]):
                p, o, row = pages[(c + i) // page], (c + i) % page, starts[b] + i
                new[p, :, o] = True
                for h in range(self.hkv):
                    e = int(scales[0][p, h, o // block]) - 127
                    if not unsure[row, h]:
                        assert e == int(self.model.scales[0][p, h, o // block]) - 127
                    y, dy = k[row, h], off[row, h]
                    got = kv8_ref.VALUES[codes[0][p, h, o]] * 2.0 ** e
                    assert np.all(np.abs(got - y) <= kv8_ref.half_step(np.abs(y) + dy, e) + dy)
        # what no call wrote, and codes that moved with a scale that both sides agree on
        same = np.repeat(scales[0] == self.model.scales[0], block, axis=2) & ~new
        assert np.array_equal(codes[0][same], self.model.codes[0][same])
        self.model.codes[0], self.model.scales[0] = codes[0].copy(), scales[0].copy()


SHAPES = [  # hq, hkv, hd, page, block
    (8, 2, 128, 16, 16), (4, 4, 64, 32, 8), (6, 6, 48, 24, 24), (2, 1, 256, 16, 4), (8, 1, 128, 64, 64), (3, 3, 16, 10, 1),
    (2, 2, 112, 256, 256), (4, 2, 128, 100, 100), (4, 2, 96, 100, 20), (5, 1, 128, 128, 128), (1, 1, 32, 7, 7)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,hd,page,block", SHAPES)
@pytest.mark.parametrize("norm,rd,interleaved", [(False, 0, False), (True, -1, False), (True, 16, True), (False, -1, True),
                                                 (True, 0, False)])
def test_calls_one_after_the_other(cuda, dtype, hq, hkv, hd, page, block, norm, rd, interleaved):
    """A prompt, then single tokens and trees behind it: blocks begun, filled and passed, with
    values that grow (scales and earlier codes move) and shrink (they stay)."""
    s = State(cuda, 3, 340, hkv, hd, page, block, dtype, seed=hd + block, rd=hd if rd < 0 else rd, interleaved=interleaved, norm=norm)
    ctx = [0, 0, 0]
    for counts, size in [([70, 3, 0], 1.0), ([1, 1, 1], 8.0), ([1, 1, 1], 0.01), ([9, 130, 2], 300.0), ([1, 0, 1], 1e-3),
                         ([2, 2, 64], 40.0)]:
        rows = sum(counts)
        sizes = [size * (1 + r % 3) for r in range(rows)]
        s.append(s.heads(rows, hq, sizes), hq, ctx, counts)
        ctx = [c + n for c, n in zip(ctx, counts)]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_drafted_slots_are_written_over(cuda, dtype):
    """A tree's slots, then the accepted tokens over them: the scale that larger drafts left
    stays until the block is begun again."""
    s = State(cuda, 1, 96, 2, 64, 32, 16, dtype, seed=5, rd=64, norm=True)
    s.append(s.heads(20, 4), 4, [0], [20])
    s.append(s.heads(10, 4, [50.0] * 10), 4, [20], [10], positions=[20, 21, 21, 22, 22, 22, 23, 23, 24, 24])
    s.append(s.heads(3, 4), 4, [20], [3])
    s.append(s.heads(40, 4), 4, [23], [40])
    s.append(s.heads(17, 4, [0.001] * 17), 4, [16], [17])  # back to a block's first slot


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_at_every_edge(cuda, dtype):
    """Zeros, the smallest and largest values, ones halfway between two codes, infinities and NaN."""
    hd = 64
    s = State(cuda, 1, 64, 1, hd, 16, 4, dtype, seed=6)
    big = torch.finfo(dtype).max
    x = torch.zeros(12, 2, hd)
    x[4:8] = torch.tensor([448.0, 432.0, 440.0, 464.0, 17.0, 19.0, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 2 ** -11, -448.0, -0.0, 1.0, 1.0625,
                           1.1875, 2 ** -6])[torch.arange(hd) % 16] * torch.tensor([1.0, 0.5, 2.0, 0.25])[:, None, None]
    x[8] = torch.where(torch.arange(hd) % 2 == 0, big, -big)
    x[9] = torch.finfo(dtype).tiny
    x[10, :, 3], x[10, :, 4], x[10, :, 5] = float("inf"), float("-inf"), float("nan")
    x[11] = 2.0 ** -45
    s.append(x.to(dtype), 0, [0], [12])
    assert s.model.scales[1][int(s.table[0, 0]), 0].tolist()[:3] == [87, 129, 167]
    # finite values beside ones that are not
    y = torch.randn(2, 2, hd, generator=s.g)
    y[:, :, 0] = float("inf")
    s.append(y.to(dtype), 0, [12], [2])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_outside_the_sequences_and_other_slots_are_left(cuda, dtype):
    s = State(cuda, 4, 64, 2, 64, 16, 8, dtype, seed=7, rd=64, norm=True)
    x = s.heads(12, 4)
    x[:2] = float("nan")
    x[9:] = float("nan")
    out = torch.full((12, 4, 64), 5.0, dtype=dtype, device=cuda)
    s.append(x, 4, [0, 13, 0, 5], [3, 0, 0, 4], lead=2, q_out=out)
    assert bool((out[:2] == 5.0).all()) and bool((out[9:] == 5.0).all())


def test_sequence_ids_and_in_place(cuda):
    s = State(cuda, 4, 64, 2, 64, 16, 16, BF16, seed=8, rd=32, norm=True)
    s.append(s.heads(9, 4), 4, [0, 17], [5, 4], seqs=[3, 1])
    x = s.heads(6, 4)
    d = x.to(cuda)
    q = ops.paged_kv8_append(d[:, :4], d[:, 4:6], d[:, 6:], s.cache, i32([5, 21], cuda), i32([0, 3, 6], cuda), 3, table=s.rope,
                             q_weight=s.wq.to(cuda), k_weight=s.wk.to(cuda), seq_ids=i32([3, 1], cuda), q_out=d[:, :4])
    want, _ = ops.qk_norm_rotary(x[:, :4].to(cuda), None, s.wq.to(cuda), None, i32([5, 6, 7, 21, 22, 23], cuda), s.rope)
    assert bits_equal(q, want) and bits_equal(d[:, 4:], x[:, 4:])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_sequences_pages_and_positions(cuda, dtype):
    s = State(cuda, 4, 64, 2, 64, 16, 16, dtype, seed=9, rd=64)
    counts, x = [3, 2, 4, 1], s.heads(10, 2)
    clean = [t.clone() for t in (s.cache.k_pages, s.cache.v_pages, s.cache.k_scales, s.cache.v_scales)]
    good = [t.clone() for t in clean]
    alone = ops.PagedKV8(*good, s.cache.page_table)
    d = x.to(cuda)

    def go(bit, bad, ctx=(0, 3, 16, 60), starts=(0, 3, 5, 9, 10), seqs=(0, 1, 2, 3), most=4, positions=None):
        for t, c in zip((s.cache.k_pages, s.cache.v_pages, s.cache.k_scales, s.cache.v_scales), clean):
            t.view(torch.uint8).copy_(c.view(torch.uint8))
        for t, c in zip(good, clean):
            t.view(torch.uint8).copy_(c.view(torch.uint8))
        st = ops.DeviceStatus(cuda)
        out = torch.full((10, 2, 64), 5.0, dtype=dtype, device=cuda)
        pos = None if positions is None else i32(positions, cuda)
        ops.paged_kv8_append(d[:, :2], d[:, 2:4], d[:, 4:], s.cache, i32(ctx, cuda), i32(starts, cuda), most, table=s.rope,
                             seq_ids=i32(seqs, cuda), positions=pos, q_out=out, status=st)
        assert st.read() == bit
        # the good ones by themselves, one call each
        for b in range(4):
            rows = slice(sum(counts[:b]), sum(counts[:b + 1]))
            if b in bad:
                assert bool((out[rows] == 5.0).all())
                continue
            q = ops.paged_kv8_append(d[rows, :2], d[rows, 2:4], d[rows, 4:], alone, i32([ctx[b]], cuda), i32([0, counts[b]], cuda), 4,
                                     table=s.rope, seq_ids=i32([seqs[b]], cuda))
            assert bits_equal(q, out[rows])
        for t, c in zip((s.cache.k_pages, s.cache.v_pages, s.cache.k_scales, s.cache.v_scales), good):
            assert torch.equal(t.view(torch.uint8), c.view(torch.uint8))

    go(0, [])
    go(_lib.BM_DEVERR_BAD_SEQUENCE, [1, 3], seqs=(0, 4, 2, -1))
    go(_lib.BM_DEVERR_BAD_POSITION, [2], ctx=(0, 3, -1, 60))
    go(_lib.BM_DEVERR_BAD_POSITION, [2], most=3)
    go(_lib.BM_DEVERR_BAD_POSITION, [3], ctx=(0, 3, 16, 64))           # behind the last page
    go(_lib.BM_DEVERR_BAD_POSITION, [3], ctx=(0, 3, 16, 2 ** 31 - 1))
    go(_lib.BM_DEVERR_BAD_POSITION, [3], starts=(0, 3, 5, 9, 11))
    go(_lib.BM_DEVERR_BAD_POSITION, [0], starts=(-1, 3, 5, 9, 10))
    # a bad page: its slots are skipped, Q is not
    page = int(s.table[1, 0])
    for bad in (-1, 10 ** 6):
        s.cache.page_table[1, 0] = bad
        st = ops.DeviceStatus(cuda)
        before = s.cache.k_pages.view(torch.uint8)[page].clone()
        ops.paged_kv8_append(None, d[:3, 2:4], d[:3, 4:], s.cache, i32([0], cuda), i32([0, 3], cuda), 3, table=s.rope,
                             seq_ids=i32([1], cuda), status=st)
        assert st.read() == _lib.BM_DEVERR_BAD_PAGE
        assert torch.equal(s.cache.k_pages.view(torch.uint8)[page], before)
    s.cache.page_table[1, 0] = page
    # positions outside the table: their rows are skipped, K, V and Q alike
    st = ops.DeviceStatus(cuda)
    out = torch.full((3, 2, 64), 5.0, dtype=dtype, device=cuda)
    before = [t.view(torch.uint8).clone() for t in (s.cache.k_pages, s.cache.v_pages)]
    ops.paged_kv8_append(d[:3, :2], d[:3, 2:4], d[:3, 4:], s.cache, i32([16], cuda), i32([0, 3], cuda), 3, table=s.rope,
                         seq_ids=i32([1], cuda), positions=i32([16, 64, 17], cuda), q_out=out, status=st)
    assert st.read() == _lib.BM_DEVERR_BAD_POSITION
    assert bool((out[1] == 5.0).all()) and not bool((out[0] == 5.0).any())
    page = int(s.table[1, 1])
    for t, b in zip((s.cache.k_pages, s.cache.v_pages), before):
        now = t.view(torch.uint8)
        assert torch.equal(now[page, :, 1], b[page, :, 1]) and not torch.equal(now[page, :, 0], b[page, :, 0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,hd,page,block", SHAPES)
def test_read(cuda, dtype, hq, hkv, hd, page, block):
    g = np.random.RandomState(hd + page)
    s = State(cuda, 5, 600, hkv, hd, page, block, dtype, seed=11)
    for codes, scales in zip(s.model.codes, s.model.scales):
        codes[:] = g.randint(0, 256, codes.shape)
        scales[:] = g.randint(80, 175, scales.shape)
    s.cache = ops.PagedKV8(*s.model.tensors(cuda), s.cache.page_table)
    first, counts, seqs = [0, 17, 599, 300, 5], [600, 33, 1, 0, 130], [0, 2, 4, 1, 2]
    starts = np.concatenate([[2], 2 + np.cumsum(counts)]).tolist()
    rows = starts[-1] + 3
    st = ops.DeviceStatus(cuda)
    outs = [torch.full((rows, hkv, hd), 5.0, dtype=dtype, device=cuda) for _ in range(2)]
    ops.paged_kv8_read(s.cache, i32(first, cuda), i32(starts, cuda), rows, 600, seq_ids=i32(seqs, cuda), k_out=outs[0],
                       v_out=outs[1], status=st)
    assert st.read() == 0
    for which, out in enumerate(outs):
        want = np.full((rows, hkv, hd), 5.0)
        values = s.model.values(which)
        for b in range(5):
            for i in range(counts[b]):
                t = first[b] + i
                want[starts[b] + i] = values[int(s.table[seqs[b], t // page]), :, t % page]
        assert np.array_equal(out.cpu().double().numpy(), want, equal_nan=True)
    made = ops.paged_kv8_read(s.cache, i32([3], cuda), i32([0, 4], cuda), 4, 4, dtype=dtype)
    assert made[0].shape == (4, hkv, hd) and made[1].dtype == dtype


def test_read_bad_sequences_and_pages(cuda):
    s = State(cuda, 3, 64, 2, 64, 16, 16, BF16, seed=12)
    s.append(s.heads(64, 0), 0, [0], [64])
    good = ops.paged_kv8_read(s.cache, i32([0], cuda), i32([0, 64], cuda), 64, 64)

    def go(first, starts, seqs, bit, kept, most=40):
        st = ops.DeviceStatus(cuda)
        outs = [torch.full((40, 2, 64), 5.0, dtype=BF16, device=cuda) for _ in range(2)]
        ops.paged_kv8_read(s.cache, i32(first, cuda), i32(starts, cuda), 40, most, seq_ids=i32(seqs, cuda), k_out=outs[0],
                           v_out=outs[1], status=st)
        assert st.read() == bit
        for out, all_ in zip(outs, good):
            for r, t in kept.items():
                assert bits_equal(out[r], all_[t])
            rest = [r for r in range(40) if r not in kept]
            assert bool((out[rest] == 5.0).all())

    go([4], [0, 40], [0], 0, {r: r + 4 for r in range(40)})
    go([4, 0], [0, 20, 40], [0, 3], _lib.BM_DEVERR_BAD_SEQUENCE, {r: r + 4 for r in range(20)})
    go([-1, 7], [0, 20, 40], [0, 0], _lib.BM_DEVERR_BAD_POSITION, {r: r - 13 for r in range(20, 40)})
    go([45, 7], [0, 20, 40], [0, 0], _lib.BM_DEVERR_BAD_POSITION, {r: r - 13 for r in range(20, 40)})
    go([4], [0, 41], [0], _lib.BM_DEVERR_BAD_POSITION, {})
    go([4], [0, 40], [0], _lib.BM_DEVERR_BAD_POSITION, {}, most=39)
    s.cache.page_table[0, 1] = 99
    go([0], [0, 40], [0], _lib.BM_DEVERR_BAD_PAGE, {r: r for r in list(range(16)) + list(range(32, 40))})


def test_streams_graphs_and_nothing_to_do(cuda):
    s = State(cuda, 3, 200, 2, 128, 16, 16, BF16, seed=13, rd=128, norm=True)
    x = s.heads(150, 4)
    s.append(x, 4, [0, 0, 0], [100, 49, 1])
    names = ("k_pages", "v_pages", "k_scales", "v_scales")
    want = [getattr(s.cache, n).view(torch.uint8).clone() for n in names]
    d = x.to(cuda)
    args = (d[:, :4], d[:, 4:6], d[:, 6:], s.cache, i32([0, 0, 0], cuda), i32([0, 100, 149, 150], cuda), 100)
    kw = dict(table=s.rope, q_weight=s.wq.to(cuda), k_weight=s.wk.to(cuda), eps=1e-4)
    first = ops.paged_kv8_append(*args, **kw)

    def wiped():
        for n in names:
            getattr(s.cache, n).view(torch.uint8).fill_(127)

    def same():
        used = [p for row, n in zip(s.table.tolist(), (100, 49, 1)) for p in row[:-(-n // 16)]]
        for n, w in zip(names, want):
            got = getattr(s.cache, n).view(torch.uint8)
            full = [p for row, c in zip(s.table.tolist(), (100, 49, 1)) for p in row[:c // 16]]
            assert torch.equal(got[full], w[full])
            if "scales" in n:
                assert torch.equal(got[used], w[used])

    side = torch.cuda.Stream()
    wiped()
    side.wait_stream(torch.cuda.current_stream())
    out = ops.paged_kv8_append(*args, **kw, stream=side)
    k, v = ops.paged_kv8_read(s.cache, i32([0, 0, 0], cuda), args[5], 150, 100, stream=side)
    side.synchronize()
    same()
    assert bits_equal(out, first)
    graph, q_out = torch.cuda.CUDAGraph(), torch.empty_like(first)
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    with torch.cuda.graph(graph):
        ops.paged_kv8_append(*args, **kw, q_out=q_out)
        ops.paged_kv8_read(s.cache, args[4], args[5], 150, 100, k_out=k2, v_out=v2)
    for _ in range(2):
        wiped()
        k2.zero_()
        graph.replay()
        same()
        assert bits_equal(q_out, first) and bits_equal(k2, k) and bits_equal(v2, v)
    none = i32([], cuda)
    ops.paged_kv8_append(None, d[:0, 4:6], d[:0, 6:], s.cache, none, i32([0], cuda), 0)
    assert ops.paged_kv8_read(s.cache, none, i32([0], cuda), 0, 0)[0].shape == (0, 2, 128)


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^31 elements from the first."""
    hkv, hd, page = 8, 128, 64
    pages = 2 ** 31 // (hkv * page * hd) + 40
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=cuda)
    k, v = (torch.zeros(pages, hkv, page, hd, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, 4, dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu) for _ in range(2))
    cache = ops.PagedKV8(k, v, ks, vs, table)
    small = ops.PagedKV8(*(torch.zeros_like(t[:2].view(torch.uint8)).view(t.dtype) for t in (k, v, ks, vs)), i32([[0, 1]], cuda))
    x = randn((100, 16, hd), BF16, gen(3)).to(cuda)
    for c in (cache, small):
        ops.paged_kv8_append(None, x[:, :8], x[:, 8:], c, i32([5], cuda), i32([0, 100], cuda), 100)
    a, b = (ops.paged_kv8_read(c, i32([5], cuda), i32([0, 100], cuda), 100, 100) for c in (cache, small))
    assert bits_equal(a[0], b[0]) and bits_equal(a[1], b[1])
    q = randn((3, 16, hd), BF16, gen(4)).to(cuda)
    outs = [ops.paged_kv8_tree_attention(q, c, i32([102], cuda), i32([0, 3], cuda), 102, 3) for c in (cache, small)]
    assert bits_equal(*outs) and bool(torch.isfinite(outs[0].float()).all())


def test_bounds_far_above_the_rows(cuda):
    """max_tokens and max_rows that bound nothing: the same codes and rows as with close ones."""
    hkv, hd, most = 2, 64, 2 ** 31 - 1
    x = randn((45, 2 * hkv + 4, hd), BF16, gen(8)).to(cuda)
    ctx, starts = i32([7, 0, 30], cuda), i32([0, 20, 21, 45], cuda)
    got = []
    for tokens, rows in ((24, 24), (most, most), (45, most)):
        s = State(cuda, 3, 70, hkv, hd, 16, 8, BF16, seed=9, rd=hd, norm=True)
        st = ops.DeviceStatus(cuda)
        q = ops.paged_kv8_append(x[:, :4], x[:, 4:4 + hkv], x[:, 4 + hkv:], s.cache, ctx, starts, tokens, table=s.rope,
                                 q_weight=s.wq.to(cuda), k_weight=s.wk.to(cuda), status=st)
        k, v = ops.paged_kv8_read(s.cache, ctx, starts, 45, rows, status=st)
        assert st.read() == 0
        got.append((q, k, v))
    for other in got[1:]:
        assert all(bits_equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("dtype,hq,hkv,hd,rd,page,block,norm", [(BF16, 8, 2, 128, 128, 64, 64, True), (BF16, 3, 1, 48, 24, 24, 8, False),
                                                                (F32, 4, 2, 64, 64, 100, 100, True), (BF16, 0, 2, 64, 0, 16, 1, False)])
def test_large_calls_write_what_small_ones_do(cuda, dtype, hq, hkv, hd, rd, page, block, norm):
    """Rows by the ten thousand, which Q, K and V have kernels of their own for, against one call a sequence."""
    rng = np.random.RandomState(hd)
    counts = [int(n) for n in rng.randint(0, 600, 50)] + [1, 1, 12287]
    ctx = [int(c) for c in rng.randint(0, 300, 50)] + [5, 0, 77]
    batch, rows, starts = len(counts), sum(counts), np.concatenate([[0], np.cumsum(counts)]).tolist()
    x = randn((rows, hq + 2 * hkv, hd), dtype, gen(hd)).to(cuda)
    got = []
    for whole in (True, False):
        s = State(cuda, batch, 12365, hkv, hd, page, block, dtype, seed=2, rd=rd, norm=norm)
        for t in (s.cache.k_scales, s.cache.v_scales):
            t.view(torch.uint8).fill_(118)
        for t in (s.cache.k_pages, s.cache.v_pages):
            t.view(torch.uint8).fill_(0x35)
        st, q_out = ops.DeviceStatus(cuda), torch.zeros((rows, hq, hd), dtype=dtype, device=cuda)
        for seqs in [range(batch)] if whole else [[b] for b in range(batch)]:
            part = slice(starts[seqs[0]], starts[seqs[-1] + 1])
            n = [counts[b] for b in seqs]
            ops.paged_kv8_append(x[part, :hq] if hq else None, x[part, hq:hq + hkv], x[part, hq + hkv:], s.cache, i32([ctx[b] for b in seqs], cuda),
                                 i32(np.concatenate([[0], np.cumsum(n)]).tolist(), cuda), max(n), table=s.rope, seq_ids=i32(list(seqs), cuda),
                                 q_weight=s.wq.to(cuda) if norm and hq else None, k_weight=s.wk.to(cuda) if norm else None,
                                 q_out=q_out[part] if hq else None, status=st)
        assert st.read() == 0
        got.append([t.view(torch.uint8) for t in (s.cache.k_pages, s.cache.v_pages, s.cache.k_scales, s.cache.v_scales)] + [q_out])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not bool((got[0][0] == 0x35).all())
