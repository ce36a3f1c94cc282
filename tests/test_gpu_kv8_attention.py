"""Tree attention over an 8-bit paged cache on the GPU against 64-bit softmax attention over the
values that the cache stands for. On the CUDA cores the tolerance is serving_ref's. On the tensor
cores queries and weights are taken in 8-bit parts. Most tests allow for a query of two e4m3 parts and for a weight
of an e5m2 and an e4m3 part of its fp16 value (a row's largest query scaled to [128, 256), its largest weight
times V's scale to 2^6 or more); the kernel's parts are closer, and Parts and the long flat contexts hold it to that.
What they add:
* a query element off by at most 2^-10 of the 128 that its row's largest exceeds, 2^-17 of that;
* a weight off by 2^-11 + 2^-8 of itself (the first part leaves at most 2^-3 of its power of two, of
  which the second loses at most 2^-5: its steps are 2^-7 up to 2^-3), or, where what is left is below the
  second part's normal range, by 2^-10, which is 2^-16 of the largest weight times scale."""
import math

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import kv8_ref, serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


def on_tensor_cores(dtype, hd, page, block):
    """Whether the header says so: bf16, heads up to 128, pages up to 128 that are multiples of 8
    or at least 64, or with an equal part of 64 to 128 slots; eight neighbouring slots of a
    tile with one scale."""
    if page <= 128:
        tile, box = (128 // page * page, page) if page % 8 == 0 else (page, page)
    else:
        parts = next(n for n in range(-(-page // 128), page + 1) if page % n == 0)
        tile = box = page // parts
    return (dtype == BF16 and hd <= 128 and tile >= 64
            and ((block % 8 == 0 and box % 8 == 0) or (tile == box and block % box == 0)))


class Batch:
    """Sequences of (context, drafted tokens) over shuffled pages. Behind each sequence's last
    slot, and in pages of nobody, codes are NaN; scales that cover none of its slots are 0 or 255."""

    def __init__(self, cuda, lens, hq, hkv, hd, page, block, dtype, seed=0, spread=2.0, extra_rows=0, tree=True, lead_rows=0,
                 exponents=(-9, -4)):
        g, rng = gen(seed), np.random.RandomState(seed)
        self.cuda, self.lens, self.page, self.block, self.dtype, self.hd, self.group = cuda, lens, page, block, dtype, hd, hq // hkv
        need = [-(-(c + n) // page) for c, n in lens]
        width = max(need + [1])
        ids = torch.randperm(sum(need) + 2, generator=g).tolist()
        table, at = [], 0
        for n in need:
            table.append(ids[at:at + n] + [-7] * (width - n))
            at += n
        self.model = kv8_ref.Cache(len(ids), hkv, page, hd, block)
        for codes, scales in zip(self.model.codes, self.model.scales):
            scales[:] = rng.choice([0, 255], scales.shape)
            for b, (c, n) in enumerate(lens):
                for p in range(need[b]):
                    slots = min(page, c + n - p * page)
                    codes[table[b][p], :, :slots] = kv8_ref.encode(rng.randn(hkv, slots, hd) * 100)
                    blocks = -(-slots // block)
                    scales[table[b][p], :, :blocks] = rng.randint(exponents[0] + 127, exponents[1] + 128, (hkv, blocks))
        self.starts = [lead_rows]
        for _, n in lens:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + extra_rows
        self.q = randn((self.rows, hq, hd), dtype, g, scale=spread)
        self.max_ctx, self.max_tree = max(c for c, _ in lens), max(n for _, n in lens)
        self.words = -(-max(self.max_tree, 1) // 64)
        self.parents = [[rng.randint(max(-1, j - 5), j) for j in range(n)] for _, n in lens]
        self.mask = torch.zeros(self.rows, self.words, dtype=torch.int64)
        for b in range(len(lens)):
            if lens[b][1]:
                self.mask[self.starts[b]:self.starts[b + 1]] = ref.tree_bits(self.parents[b], self.words)
        self.tree = tree
        self.table = torch.tensor(table, dtype=torch.int32)
        self.tc = on_tensor_cores(dtype, hd, page, block)
        self.upload()

    def upload(self):
        self.cache = ops.PagedKV8(*self.model.tensors(self.cuda), self.table.to(self.cuda))

    def args(self):
        return (self.q.to(self.cuda), self.cache, i32([c for c, _ in self.lens], self.cuda), i32(self.starts, self.cuda),
                self.max_ctx, self.max_tree)

    def run(self, **kw):
        return ops.paged_kv8_tree_attention(*self.args(), **{**dict(tree_mask=self.mask.to(self.cuda) if self.tree else None), **kw})

    def want(self, scale=None, seqs=None):
        bits = self.mask.numpy().view(np.uint64)
        if self.tree:
            mask = lambda row, i, j: bool((int(bits[row, j // 64]) >> (j % 64)) & 1)  # noqa: E731
        else:
            mask = lambda row, i, j: j <= i  # noqa: E731
        k, v = (torch.from_numpy(np.nan_to_num(self.model.values(w))) for w in range(2))
        seqs = seqs or list(range(len(self.lens)))
        scale = scale or 1 / math.sqrt(self.hd)
        out, tol = ref.attention(self.q, k, v, self.table, seqs, [c for c, _ in self.lens], self.starts, mask, scale, self.dtype, self.tc)
        if self.tc:
            tol += 1.05 * self.parts(k, v, seqs, mask, scale)
        return out, tol

    def parts(self, k, v, seqs, mask, scale):
        """The tensor cores' part of the tolerance, as the module's comment derives it."""
        extra = np.zeros(self.q.shape)
        vs = 2.0 ** (np.clip(self.model.scales[1].astype(np.int64), 87, 167) - 127.0)
        q = self.q.double().numpy()
        for b, (c, n) in enumerate(self.lens):
            if n == 0:
                continue
            slots = np.arange(c + n)
            ids, off = self.table[seqs[b]].numpy()[slots // self.page], slots % self.page
            seen = np.ones((n, c + n), dtype=bool)
            for i in range(n):
                seen[i, c:] = [mask(self.starts[b] + i, i, j) for j in range(n)]
            for h in range(q.shape[1]):
                kv, rows = h // self.group, slice(self.starts[b], self.starts[b + 1])
                kh, vh, ve = k[ids, kv, off].numpy(), np.abs(v[ids, kv, off].numpy()), vs[ids, kv, off // self.block]
                x = q[rows, h]
                s = np.where(seen, x @ kh.T * scale, -np.inf)
                top = s.max(-1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
                size = np.where(seen, np.abs(kh).sum(-1), 0.0).max(-1)
                ds = 2.0 ** -17 * np.abs(x).max(-1) * size * scale
                total = np.where(seen.any(-1), p.sum(-1), 1.0)
                extra[rows, h] = ((2 * ds + 2.0 ** -11)[:, None] * (p @ vh)
                                  + 2.0 ** -16 * (p * ve).max(-1)[:, None] * (seen @ (vh / ve[:, None]))) / total[:, None]
        return extra

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


def test_which_cores():
    """The shapes below reach both."""
    takes = [on_tensor_cores(*s) for s in ((BF16, 128, 16, 16), (BF16, 48, 16, 8), (BF16, 128, 100, 100), (BF16, 64, 200, 200),
                                           (BF16, 128, 256, 8), (BF16, 128, 512, 64))]
    lacks = [on_tensor_cores(*s) for s in ((F32, 128, 16, 16), (BF16, 256, 16, 16), (BF16, 128, 16, 4), (BF16, 128, 100, 20),
                                           (BF16, 128, 136, 8), (BF16, 128, 7, 7))]
    assert all(takes) and not any(lacks)


@pytest.mark.parametrize("dtype,hq,hkv,hd,page,block", [
    (BF16, 8, 2, 128, 16, 16), (BF16, 4, 4, 128, 64, 64), (BF16, 16, 2, 128, 8, 8), (BF16, 7, 1, 128, 128, 32), (BF16, 8, 1, 64, 32, 8),
    (BF16, 6, 2, 64, 256, 256), (BF16, 4, 2, 128, 24, 24), (BF16, 4, 2, 48, 16, 8), (BF16, 24, 2, 128, 512, 64),
    (BF16, 4, 2, 80, 100, 100), (BF16, 8, 1, 16, 72, 72), (BF16, 3, 1, 112, 200, 200), (BF16, 32, 1, 112, 24, 8),
    (BF16, 4, 2, 128, 250, 250),
    (BF16, 2, 1, 256, 16, 16), (BF16, 4, 1, 96, 7, 7), (BF16, 8, 2, 128, 16, 4), (BF16, 4, 2, 64, 100, 20), (BF16, 2, 1, 128, 136, 8),
    (F32, 6, 6, 48, 16, 16), (F32, 8, 2, 128, 7, 1), (F32, 4, 1, 256, 100, 50), (F32, 2, 2, 16, 1, 1), (F32, 6, 1, 96, 32, 4)])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("tree", [True, False])
def test_against_64_bits(cuda, lens, dtype, hq, hkv, hd, page, block, tree):
    Batch(cuda, LENS[lens], hq, hkv, hd, page, block, dtype, seed=hd + page, tree=tree).check()


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (BF16, 64), (F32, 48), (BF16, 80), (BF16, 256)])
def test_many_uneven_sequences(cuda, dtype, hd):
    rng = np.random.RandomState(3)
    lens = [(int(rng.randint(0, 600)), int(rng.randint(0, 12))) for _ in range(70)]
    Batch(cuda, lens, 4, 2, hd, 16, 16, dtype, seed=4).check()


@pytest.mark.parametrize("hq,hkv,hd,page,block", [
    (8, 2, 128, 16, 16), (8, 2, 64, 32, 1), (4, 4, 48, 24, 3), (32, 1, 128, 64, 64), (20, 1, 112, 128, 2), (7, 7, 16, 8, 8),
    (5, 1, 80, 100, 50), (3, 1, 128, 256, 128), (11, 1, 96, 200, 25), (64, 1, 128, 16, 16), (33, 1, 64, 16, 8)])
@pytest.mark.parametrize("rows", [1, 8, 9, 31, 32, 33, 48, 64, 65, 127, 128, 129, 256, 257])
def test_rows_about_every_form(cuda, hq, hkv, hd, page, block, rows):
    """Trees whose rows (tokens times group) fill, and pass, the tiles of 32, 64, 128 and 256 rows."""
    n = max(1, rows // (hq // hkv))
    Batch(cuda, [(700, n), (0, n), (131, max(1, n - 1)), (40, 1)], hq, hkv, hd, page, block, BF16, seed=rows + hd).check()


@pytest.mark.parametrize("hq,hkv,most", [(8, 2, 4), (6, 3, 24), (8, 1, 16), (16, 2, 40)])
@pytest.mark.parametrize("seed", range(4))
def test_cuts_anywhere_about_short_items(cuda, hq, hkv, most, seed):
    """One long context among many short ones: shares of the work begin and end in items of one
    tile, at their borders, and in what an item's beginning counts for."""
    rng = np.random.RandomState(seed)
    lens = [(int(rng.choice([0, 1, 100, 128, 129, 300])), int(rng.randint(0, most + 1))) for _ in range(45 + seed)]
    lens[int(rng.randint(len(lens)))] = (2000 + 300 * seed, most)
    Batch(cuda, lens, hq, hkv, 64, 16, 16, BF16, seed=seed, tree=seed != 2).check()


@pytest.mark.parametrize("group,most,batch", [(4, 8, 256), (4, 16, 128), (8, 16, 128), (8, 40, 64)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("mixed", [False, True])
def test_many_short_items_in_every_form(cuda, group, most, batch, hd, mixed):
    """Items by far more than CTAs: runs of segments of one tile, between longer ones when mixed,
    in the forms of 32, 64, 128 and 256 rows. Twice over with the same bits."""
    rng = np.random.RandomState(batch + most)
    lens = [(int(rng.randint(300, 601) if mixed and rng.rand() < 0.2 else rng.randint(0, 121)), int(rng.randint(1, most + 1)))
            for _ in range(batch)]
    lens[0] = (lens[0][0], most)
    b = Batch(cuda, lens, 8 * group, 8, hd, 16, 16, BF16, seed=most + hd)
    first = b.check()
    for _ in range(3):
        assert bits_equal(b.run(), first)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_wide_groups(cuda, dtype):
    Batch(cuda, [(200, 3), (9, 30)], 64, 1, 128, 32, 32, dtype, seed=5).check()
    Batch(cuda, [(200, 9)], 33, 1, 64, 32, 8, dtype, seed=6).check()


@pytest.mark.parametrize("dtype,hd,page,block", [(BF16, 128, 16, 16), (F32, 64, 10, 5), (BF16, 48, 16, 8), (BF16, 256, 16, 16)])
def test_rows_that_see_little_or_nothing(cuda, dtype, hd, page, block):
    """Masks that leave a row empty (zeros), hide a row from itself, and set bits past the tree."""
    b = Batch(cuda, [(0, 4), (0, 70), (130, 3), (5, 2)], 4, 2, hd, page, block, dtype, seed=7)
    b.mask[0] = 0
    b.mask[1] = -1  # every bit, those past the tree too
    b.mask[2] = 1 << 3
    b.mask[10] = 0
    b.mask[b.starts[2]] = 0
    b.mask[b.starts[3] + 1] = torch.tensor([-4, -1])
    got = b.check()
    assert int(torch.count_nonzero(got[0])) == 0 and int(torch.count_nonzero(got[10])) == 0


@pytest.mark.parametrize("dtype,hd,block", [(BF16, 128, 16), (BF16, 64, 8), (F32, 48, 4), (BF16, 128, 2)])
@pytest.mark.parametrize("exponents", [(-40, 40), (-40, -39), (39, 40), (-30, -10), (0, 20)])
def test_scales_far_apart(cuda, dtype, hd, block, exponents):
    """Blocks whose scales differ by up to 2^80: large values of small weight next to small ones of
    large weight. Queries are small enough for scores to stay apart by little."""
    b = Batch(cuda, [(700, 2), (300, 1), (20, 40)], 4, 2, hd, 16, block, dtype, seed=23, exponents=exponents, spread=2.0 ** -10)
    b.model.scales[0][:] = np.where((b.model.scales[0] > 0) & (b.model.scales[0] < 255), 127, b.model.scales[0])
    b.upload()
    b.check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_keys_of_every_size(cuda, dtype):
    b = Batch(cuda, [(700, 2), (300, 1)], 4, 2, 128, 16, 8, dtype, seed=24, exponents=(-40, -2), spread=0.5)
    b.model.scales[1][:] = np.where((b.model.scales[1] > 0) & (b.model.scales[1] < 255), 120, b.model.scales[1])
    b.upload()
    b.check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_far_apart(cuda, dtype):
    """Maxima that rise by a lot, late and early: weights under- and overflow unless the running
    maximum follows."""
    Batch(cuda, [(700, 2), (300, 1)], 4, 2, 128, 16, 16, dtype, seed=11, spread=60.0).check()


@pytest.mark.parametrize("group,tokens", [(4, 1), (4, 12), (8, 16), (8, 40)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("slots,below,spread", [(8192, 12.83, 0.0), (8192, 13.0, 0.1), (8192, 13.0, 0.3), (8192, 13.0, 1.0),
                                                (8192, 14.83, 0.0), (131072, 17.3, 0.0), (131072, 18.0, 0.2)])
def test_one_heavy_slot_before_a_long_flat_context(cuda, group, tokens, hd, slots, below, spread):
    """The first slot's score is `below` (base 2) above those of all others, which lie within `spread` of
    each other: every weight is small, and their sum is not. As many sequences (of the same pages) as there are SMs, so
    that a CTA walks one from its first slot to its last. A weight may be off by its fp16 value's half step, 2^-11 of
    itself, so the output by that part of the sum of weights times |v|. Another half of it is for the rest:
    scores in fp32 (a few 2^-19 of a weight) and the parts' least step, 2^-17 under a lift of 2^12, which
    2^17 slots of |v| up to twice the first's make 2^-11 of that sum at the very most, and 2^-12 at random."""
    g = gen(slots + tokens)
    page, ctx = 64, slots - tokens
    pages, batch = slots // page, torch.cuda.get_device_properties(cuda).multi_processor_count
    k = torch.zeros(pages * page, hd)
    k[:, 1] = (torch.rand(pages * page, generator=g) * 2 - 1) * 16
    k[0, 0], k[0, 1] = 16.0, 0.0
    v = 64.0 * (1 + torch.rand(pages * page, hd, generator=g))
    v[0] = -v[0]  # the first slot and the others pull apart
    codes = [x.to(torch.float8_e4m3fn) for x in (k, v)]
    scales = [torch.full((pages, 1, 2), 127, dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu) for _ in range(2)]
    cache = ops.PagedKV8(*(x.to(cuda).view(pages, 1, page, hd) for x in codes), *scales,
                         torch.arange(pages, dtype=torch.int32, device=cuda).repeat(batch, 1))
    q = torch.zeros(batch * tokens, group, hd, dtype=BF16)
    q[..., 0], q[..., 1] = 2.0, spread / below
    scale = below * math.log(2.0) / 32
    st = ops.DeviceStatus(cuda)
    got = ops.paged_kv8_tree_attention(q.to(cuda), cache, i32([ctx] * batch, cuda), i32(range(0, batch * tokens + 1, tokens), cuda), ctx,
                                       tokens, scale=scale, status=st)
    assert st.read() == 0
    got = got.view(batch, tokens, group, hd)
    kd, vd = (x.double() for x in codes)
    s = (kd @ q[0, 0].double()) * float(np.float32(scale))
    for i in {0, tokens - 1}:
        p = torch.exp(s[:ctx + i + 1] - s[0])
        p /= p.sum()
        want, size = p @ vd[:ctx + i + 1], p @ vd[:ctx + i + 1].abs()
        err = (got[:, i].cpu().double() - want).abs()
        assert torch.all(err <= 1.5 * 2.0 ** -11 * size + 1.01 * ref.HALF[BF16] * want.abs()), (err / size).max()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_queries_of_every_size(cuda, dtype):
    """Heads of zeros, of tiny and of large elements, and one element far above the others."""
    b = Batch(cuda, [(200, 4), (30, 3)], 4, 2, 128, 16, 16, dtype, seed=25)
    b.q[0, 0] = 0.0
    b.q[1, 1] *= 2.0 ** -30
    b.q[2, 2] *= 2.0 ** 6
    b.q[3, 3, 5] = 100.0
    b.q[4] *= 2.0 ** -120
    b.q[5, :, ::2] *= 2.0 ** -8
    b.check()


def test_a_query_that_is_not_finite_spoils_its_row_alone(cuda):
    for dtype, block in ((BF16, 16), (BF16, 4), (F32, 16)):
        b = Batch(cuda, [(200, 4), (30, 3)], 4, 2, 128, 16, block, dtype, seed=26)
        want = b.check()
        b.q[1, 2, 7] = float("nan")
        b.q[5, 0, 3] = float("inf")
        got = b.run()
        bad = torch.zeros(b.rows, 4, dtype=torch.bool)
        bad[1, 2] = bad[5, 0] = True
        assert torch.isnan(got.cpu()[bad]).all()
        assert bits_equal(got.cpu()[~bad], want.cpu()[~bad])


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_rows_outside_the_sequences_are_left(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (300, 2)], 4, 2, hd, 16, 16, dtype, seed=8, extra_rows=4, lead_rows=2)
    b.q[:2] = float("nan")
    out = torch.full((b.rows, 4, hd), 5.0, dtype=dtype, device=cuda)
    b.check(b.run(out=out))
    keep = torch.full_like(out[0], 5.0)
    for r in [0, 1] + list(range(b.starts[-1], b.rows)):
        assert bits_equal(out[r], keep)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_bad_sequences_are_skipped_and_others_served(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (300, 2), (17, 4), (64, 1)], 4, 2, hd, 16, 16, dtype, seed=9)
    want, tol = b.want()

    def go(ctx, starts, seqs, bit, bad, max_ctx=300, max_tree=4):
        out, st = torch.full((b.rows, 4, hd), 5.0, dtype=dtype, device=cuda), ops.DeviceStatus(cuda)
        ops.paged_kv8_tree_attention(b.q.to(cuda), b.cache, i32(ctx, cuda), i32(starts, cuda), max_ctx, max_tree,
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
    go([40, 303, 17, 64], st, [0, 1, 2, 3], _lib.BM_DEVERR_BAD_POSITION, [1], max_ctx=400)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_a_bad_page_is_flagged_and_unseen(cuda, dtype, hd):
    b = Batch(cuda, [(100, 2)], 4, 2, hd, 16, 16, dtype, seed=10)
    k, v = (np.nan_to_num(b.model.values(w))[b.table[0].numpy()].transpose(1, 0, 2, 3).reshape(2, -1, hd)[:, :102] for w in range(2))
    s = np.einsum("hd,sd->hs", b.q[0, :2].double().numpy(), k[0]) / math.sqrt(hd)
    s[:, 32:48] = -np.inf  # the page's slots are left out of the softmax
    s[:, 101] = -np.inf    # row 0 does not see slot 1
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = p @ v[0]
    # weights and output rounded to the type (2^-11 for a weight's parts), half a step each
    tol = 1.01 * (ref.HALF[dtype] + 2.0 ** -11) * (p @ np.abs(v[0]) + np.abs(want)) + 2.0 ** -15 * np.abs(v[0]).sum(0)
    for page in (-1, 10 ** 6):
        b.cache.page_table[0, 2] = page
        st = ops.DeviceStatus(cuda)
        out = b.run(status=st)
        assert st.read() == _lib.BM_DEVERR_BAD_PAGE
        assert np.all(np.abs(out[0, :2].cpu().double().numpy() - want) <= tol)


def test_sequence_ids_share_a_cache_and_scale(cuda):
    b = Batch(cuda, [(50, 2), (90, 3)], 4, 2, 128, 16, 16, BF16, seed=12)
    got = b.run(scale=0.03, seq_ids=i32([0, 1], cuda))
    want, tol = b.want(scale=0.03)
    assert np.all(np.abs(got.cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (BF16, 64), (BF16, 256), (F32, 48), (F32, 128)])
@pytest.mark.parametrize("seqs", [[3, 2, 1, 0], [1, 0, 1, 2], [2, 2, 2, 2]])
def test_sequence_ids_in_any_order_and_twice(cuda, dtype, hd, seqs):
    b = Batch(cuda, [(60, 3), (60, 3), (60, 3), (60, 3)], 8, 2, hd, 16, 16, dtype, seed=21)
    st = ops.DeviceStatus(cuda)
    got = b.run(seq_ids=i32(seqs, cuda), status=st)
    assert st.read() == 0
    want, tol = b.want(seqs=seqs)
    assert np.all(np.abs(got.cpu().double().numpy() - want) <= tol)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (F32, 48)])
def test_repeats_streams_graphs_and_dirty_workspaces(cuda, dtype, hd):
    b = Batch(cuda, [(40, 3), (1500, 2), (17, 4), (640, 1)], 4, 2, hd, 16, 16, dtype, seed=13)
    first = b.check()
    q, cache, ctx, starts, max_ctx, max_tree = b.args()
    ws = ops.paged_kv8_tree_attention_workspace(q, cache, 4, max_ctx, max_tree)
    for fill in (0xFF, 0x7F, 0):
        ws.fill_(fill)
        assert bits_equal(b.run(workspace=ws), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = b.run(stream=side)
    side.synchronize()
    assert bits_equal(out, first)
    mask = b.mask.to(cuda)
    graph, o1, o2 = torch.cuda.CUDAGraph(), torch.empty_like(q), torch.empty_like(q)
    with torch.cuda.graph(graph):
        for o in (o1, o2):
            ops.paged_kv8_tree_attention(q, cache, ctx, starts, max_ctx, max_tree, tree_mask=mask, out=o, workspace=ws)
    for _ in range(3):
        o1.zero_()
        o2.zero_()
        graph.replay()
        assert bits_equal(o1, first) and bits_equal(o2, first)
    ctx.copy_(i32([40, 700, 17, 0], cuda))  # a replay reads the lengths of its time
    graph.replay()
    want = ops.paged_kv8_tree_attention(q, cache, ctx, starts, max_ctx, max_tree, tree_mask=mask)
    assert bits_equal(o1, want) and not bits_equal(o1, first)


def test_long_prompt_chunk(cuda):
    """Hundreds of tokens behind cached ones, no mask: many row tiles per sequence."""
    Batch(cuda, [(100, 400), (3, 90)], 4, 2, 128, 16, 16, BF16, seed=15, tree=False).check()
    Batch(cuda, [(100, 300)], 4, 2, 64, 16, 16, F32, seed=16, tree=False).check()


def test_nothing_to_do(cuda):
    b = Batch(cuda, [(5, 1)], 4, 2, 128, 16, 16, BF16)
    none = i32([], cuda)
    out = ops.paged_kv8_tree_attention(b.q[:0].to(cuda), b.cache, none, i32([0], cuda), 0, 0)
    assert out.shape == (0, 4, 128)
    out = torch.full((3, 4, 128), 5.0, dtype=BF16, device=cuda)
    ops.paged_kv8_tree_attention(torch.zeros_like(out), b.cache, i32([5], cuda), i32([1, 1], cuda), 8, 4, out=out)
    assert bool((out == 5.0).all())


def test_streams_at_once(cuda):
    """Calls that overlap on the GPU, a workspace each: the same results as one after the other."""
    batches = [Batch(cuda, [(3000, 3), (1500, 2), (17, 4)], 8, 2, 128, 16, 16, BF16, seed=17),
               Batch(cuda, [(900, 30), (2000, 5)], 8, 2, 64, 32, 8, BF16, seed=18),
               Batch(cuda, [(700, 4), (90, 9)], 4, 2, 48, 16, 4, F32, seed=19)]
    first = [b.run() for b in batches]
    calls = []
    for b in batches:
        args = b.args()
        kw = [dict(tree_mask=b.mask.to(cuda), out=torch.empty_like(args[0]),
                   workspace=ops.paged_kv8_tree_attention_workspace(args[0], b.cache, len(b.lens), b.max_ctx, b.max_tree))
              for _ in range(3)]
        calls.append((args, kw))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for turn in range(10):
        for s, stream in enumerate(streams):
            for i in range(3):
                args, kw = calls[(s + i) % 3]
                ops.paged_kv8_tree_attention(*args, stream=stream, **kw[s])
    torch.cuda.synchronize()
    for (args, kw), want in zip(calls, first):
        for k in kw:
            assert bits_equal(k["out"], want)


class Parts(Batch):
    """The tensor cores' own bounds, in place of bf16 weights and of the looser ones above:
    * a query element's e4m3 part leaves at most 2^-4 of its power of two, in units of 2^-7 of it (bf16 has 8 bits): at
      most 8 of them, a number of three bits, which the e5m2 part holds. Below 2^-6 (the row's largest is scaled to
      128 at least) the first part leaves up to 2^-10, of which the second loses half a step, 2^-14: 2^-21 of 128;
    * a weight is its fp16 value, off by 2^-11 of itself at most, in parts that hold all of it or end at 2^-16, off by
      2^-17, where the largest weight times V's scale is 2^12 or more: 2^-29 of that."""

    def want(self, scale=None, seqs=None):
        assert self.tc and not self.tree and scale is None and seqs is None
        k, v = (torch.from_numpy(np.nan_to_num(self.model.values(w))) for w in range(2))
        seqs, scale = list(range(len(self.lens))), 1 / math.sqrt(self.hd)
        mask = lambda row, i, j: j <= i  # noqa: E731
        out, tol = ref.attention(self.q, k, v, self.table, seqs, [c for c, _ in self.lens], self.starts, mask, scale, self.dtype, False)
        vs = 2.0 ** (np.clip(self.model.scales[1].astype(np.int64), 87, 167) - 127.0)
        for b, (c, n) in enumerate(self.lens):
            slots = np.arange(c + n)
            ids, off = self.table[b].numpy()[slots // self.page], slots % self.page
            seen = slots[None] <= c + np.arange(n)[:, None]
            rows = slice(self.starts[b], self.starts[b + 1])
            for h in range(self.q.shape[1]):
                kv, x = h // self.group, self.q[rows, h].double().numpy()
                kh, vh, ve = k[ids, kv, off].numpy(), np.abs(v[ids, kv, off].numpy()), vs[ids, kv, off // self.block]
                s = np.where(seen, x @ kh.T * scale, -np.inf)
                p = np.exp(s - s.max(-1, keepdims=True))
                ds = 2.0 ** -21 * np.abs(x).max(-1) * np.where(seen, np.abs(kh).sum(-1), 0.0).max(-1) * scale
                extra = (2 * ds + 2.0 ** -11)[:, None] * (p @ vh) + 2.0 ** -29 * (p * ve).max(-1)[:, None] * (seen @ (vh / ve[:, None]))
                tol[rows, h] += 1.05 * extra / p.sum(-1, keepdims=True)
        return out, tol


@pytest.mark.parametrize("group,most", [(4, 8), (4, 16), (8, 16), (8, 40)])
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("above", [0, 4, 8, 12])
def test_queries_with_one_element_far_above_the_others(cuda, group, most, hd, above):
    """2^above times as large, at a place where keys are zero: the others make the scores."""
    b = Parts(cuda, [(700, most), (131, 1), (0, most)], 2 * group, 2, hd, 16, 16, BF16, seed=above + hd, tree=False)
    codes = b.model.codes[0]
    codes[..., 5] = np.where(codes[..., 5] == 127, 127, 0)
    b.q[..., 5] = 2.0 ** above
    b.upload()
    b.check()
