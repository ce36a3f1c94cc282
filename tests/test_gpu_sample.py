"""Sampling on the GPU: every token equals the 64-bit row-by-row form's."""
import math

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import serving_ref as ref
from tests.helpers import gen

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def settings(rows, g, which):
    pick = lambda values: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=g)]  # noqa: E731
    out = dict(temperature=None, top_k=None, top_p=None, min_p=None)
    if "t" in which:
        out["temperature"] = pick([0.0, 0.3, 0.7, 1.0, 1.5])
    if "k" in which:
        out["top_k"] = pick([0, 1, 3, 40, 700, -5, 10 ** 9]).to(torch.int32)
    if "p" in which:
        out["top_p"] = pick([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.5, -1.0])
    if "m" in which:
        out["min_p"] = pick([0.0, 0.001, 0.05, 0.5, 1.0, 2.0, -1.0])
    return out


def check(cuda, x, u, s):
    st = ops.DeviceStatus(cuda)
    dev = {n: None if t is None else t.to(cuda) for n, t in s.items()}
    got = ops.sample(x.to(cuda), u.to(cuda), status=st, **dev)
    assert st.read() == 0
    want = ref.sample(x, u, **s)
    assert got.cpu().tolist() == want
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", ["", "t", "tk", "tp", "tm", "tkp", "tkpm"])
@pytest.mark.parametrize("rows,vocab", [(40, 1), (40, 2), (40, 7), (60, 33), (30, 1000), (20, 5003), (8, 32000), (3, 128256)])
def test_settings_and_sizes(cuda, rows, vocab, which, dtype):
    g = gen(vocab + rows)
    spread = torch.tensor([0.05, 0.5, 1.0, 3.0, 8.0])[torch.arange(rows) % 5][:, None]
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
    check(cuda, x, torch.rand(rows, generator=g), settings(rows, g, which))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("which", ["", "tkpm"])
@pytest.mark.parametrize("values", [[0.0], [1.0, 1.0, 2.0], [-0.0, 0.0, -1.0], [5.0, -math.inf], [3.0, -3.0e38, 2.0],
                                    [-3.38e38], [3e38, -3e38, 2.9e38], [1e-40, 0.0, -1e-40]])
def test_ties_zeros_and_extremes(cuda, values, which, dtype):
    """Few values many times over: ties at every border go to the lowest index."""
    g = gen(len(values))
    for vocab in (5, 777, 9001):
        x = torch.tensor(values)[torch.randint(0, len(values), (50, vocab), generator=g)].to(dtype)
        x[x.isinf()] = -math.inf
        check(cuda, x, torch.rand(50, generator=g), settings(50, g, which))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_infinities_nan_and_rows_of_nothing(cuda, dtype):
    inf, nan = math.inf, math.nan
    rows = [[-inf] * 6, [nan] * 6, [nan, -inf, -inf, nan, -inf, nan], [-inf, -inf, 1.0, -inf, -inf, -inf],
            [nan, 2.0, 1.0, nan, -inf, 0.0], [inf, 1.0, inf, nan, -inf, inf], [inf, inf, inf, inf, inf, inf],
            [-inf, inf, 3.0, 4.0, 5.0, 6.0]]
    g = gen(3)
    x = torch.tensor(rows).to(dtype).repeat(30, 1)
    n = x.shape[0]
    got = check(cuda, x, torch.rand(n, generator=g), settings(n, g, "tkpm")).view(30, 8)
    assert bool((got[:, :3] == -1).all()) and bool((got[:, 3] == 2).all()) and bool((got[:, 7] == 1).all())


def test_uniform_borders(cuda):
    """Equal weights: token floor(u * vocab), also for u that fall on a border."""
    vocab = 1 << 12
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 2.0 ** -12, 2.0 ** -12 - 2.0 ** -24, 2.0 ** -40])
    x = torch.zeros(8, vocab)
    assert check(cuda, x, u, settings(8, gen(0), "")).tolist() == [0, 1024, 2048, 3 * 1024, 4095, 1, 0, 0]
    half = dict(settings(8, gen(0), ""), top_p=torch.full((8,), 0.5))
    assert check(cuda, x, u, half).tolist() == [0, 512, 1024, 1536, 2047, 0, 0, 0]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_temperatures_at_their_ends(cuda, dtype):
    g = gen(4)
    x = (torch.randn(12, 900, generator=g) * 3).to(dtype)
    x[:, 5] = -math.inf
    t = torch.tensor([0.0, 1e-45, 1e-30, 1e-6, 1e-3, 1e3, 1e30, math.inf, 0.0, 2.0, math.inf, 1.0])
    check(cuda, x, torch.rand(12, generator=g), dict(temperature=t, top_k=None, top_p=None, min_p=None))


def test_bad_settings_are_flagged(cuda):
    nan = math.nan
    ok = dict(temperature=[1.0] * 4, top_p=[0.9] * 4, min_p=[0.0] * 4, uniforms=[0.5] * 4)
    x = torch.tensor([[0.0, 9.0, 0.0]]).repeat(4, 1).to(cuda)
    for name, bads in (("temperature", [nan, -1.0, -math.inf]), ("top_p", [nan]), ("min_p", [nan]),
                       ("uniforms", [nan, -0.1, 1.0, math.inf])):
        for bad in bads:
            s = {n: torch.tensor(v, device=cuda) for n, v in ok.items()}
            s[name][2] = bad
            st = ops.DeviceStatus(cuda)
            got = ops.sample(x, status=st, **s)
            assert st.read() == _lib.BM_DEVERR_BAD_PARAMETER
            assert got.tolist() == [1, 1, -1, 1]


def test_strides_streams_graphs_and_no_rows(cuda):
    g = gen(5)
    for dtype in (F32, BF16):
        wide = (torch.randn(9, 2003, generator=g) * 2).to(dtype).to(cuda)
        u = torch.rand(9, generator=g)
        s = settings(9, g, "tkpm")
        dev = {n: t.to(cuda) for n, t in s.items()}
        for lo, hi in ((0, 2000), (1, 1998), (7, 8)):
            part = wide[:, lo:hi]
            want = ref.sample(part, u, **s)
            assert ops.sample(part, u.to(cuda), **dev).tolist() == want
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = ops.sample(wide, u.to(cuda), stream=side, **dev)
        side.synchronize()
        want = ref.sample(wide, u, **s)
        assert got.tolist() == want
        graph, out, ud = torch.cuda.CUDAGraph(), torch.empty(9, dtype=torch.int32, device=cuda), u.to(cuda)
        with torch.cuda.graph(graph):
            ops.sample(wide, ud, out=out, **dev)
        for _ in range(2):
            out.fill_(-9)
            graph.replay()
            assert out.tolist() == want
    assert ops.sample(torch.empty(0, 10, device=cuda), torch.empty(0, device=cuda)).shape == (0,)


def test_many_rows_and_a_large_vocabulary(cuda):
    g = gen(6)
    x = torch.randn(700, 900, generator=g) * 2
    check(cuda, x, torch.rand(700, generator=g), settings(700, g, "tkpm"))
    x = torch.randn(2, 700001, generator=g) * 2
    check(cuda, x, torch.rand(2, generator=g), dict(settings(2, g, ""), top_p=torch.tensor([0.9, 1.0])))
    check(cuda, x, torch.rand(2, generator=g), dict(settings(2, g, ""), top_k=torch.tensor([50, 5000], dtype=torch.int32)))


def test_frequencies_follow_the_weights(cuda):
    """50000 stratified numbers over one row: every token's share is its probability to
    one stratum at each of its borders."""
    n = 50000
    row = torch.tensor([1.0, -2.0, 0.5, 3.0, 3.0, -math.inf, 0.0])
    u = (torch.arange(n) + 0.5) / n
    got = ops.sample(row.expand(n, 7).contiguous().to(cuda), u.to(cuda)).cpu().long()
    p = torch.softmax(row.double(), 0)
    assert bool(((torch.bincount(got, minlength=7) / n - p).abs() <= 2.0 / n).all())


@pytest.mark.parametrize("which", ["tp", "tkp"])
def test_many_rows_at_once_and_again(cuda, which):
    """More rows than SMs (two CTAs on each), with equal logits at the borders: the same
    tokens every time."""
    g = gen(11)
    rows, vocab = 250, 128000
    x = (torch.randn(rows, vocab, generator=g) * 2.0).to(BF16)
    u = torch.rand(rows, generator=g)
    s = dict(temperature=0.7 + torch.rand(rows, generator=g), top_k=None, top_p=0.5 + 0.49 * torch.rand(rows, generator=g),
             min_p=None)
    if "k" in which:
        s["top_k"] = torch.randint(1100, 90000, (rows,), generator=g).to(torch.int32)
    got = check(cuda, x, u, s)
    dev = {n: None if t is None else t.to(cuda) for n, t in s.items()}
    x, u = x.to(cuda), u.to(cuda)
    for _ in range(30):
        assert torch.equal(ops.sample(x, u, **dev), got)


def test_ties_between_two_bins_of_the_histogram(cuda):
    """Equal logits at the border of top-p whose place in the histogram lies half way
    between two bins, but for its rounding: all of them fall into the same one."""
    g = np.random.default_rng(12)
    vocab, rows, top, ties = 2100, 160, np.float32(8.0), 100
    values = torch.arange(-4.0, 4.0, 2.0 ** -6).to(BF16).float().numpy()
    bins_per_octave = np.float32(np.float32(4094.5) / np.float32(min(51, 62 - 12) + 2))
    found = []
    while len(found) < rows:
        t = np.float32(g.uniform(0.5, 2.0))
        bins = np.float32(1.4426950408889634074 / np.float64(t) * np.float64(bins_per_octave))
        exact = (np.float64(top) - values) * np.float64(bins)
        place = exact.astype(np.float32)
        for i in np.flatnonzero((place % 1 == 0.5) & (exact != place))[:1]:
            found.append((t, values[i]))
    x = np.full((rows, vocab), -30.0, dtype=np.float32)
    p = np.empty(rows)
    for r, (t, v) in enumerate(found):
        at = g.permutation(vocab)
        x[r, at[0]], x[r, at[1:1 + ties]] = top, v
        w = np.exp((np.float64(v) - 8.0) / t)
        x[r, at[1 + ties:1 + 2 * ties]] = v - 0.5  # and less of what goes
        p[r] = (1 + w * (ties // 2 + 0.4)) / np.exp((x[r].astype(np.float64) - 8.0) / t).sum()
    s = dict(temperature=torch.tensor([float(t) for t, _ in found]), top_k=None, top_p=torch.tensor(p).float(), min_p=None)
    for u in (0.999, 0.9999, 1 - 2.0 ** -24):
        check(cuda, torch.from_numpy(x).to(BF16), torch.full((rows,), u), s)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1025, 5000, 40000])
def test_infinities_and_temperatures_of_long_rows(cuda, vocab, dtype):
    """The edges of the settings where a row is shared by warps or CTAs."""
    inf, nan = math.inf, math.nan
    g = gen(vocab)
    heads = [[-inf] * 6, [nan] * 6, [nan, -inf, 1.0, nan, -inf, -inf], [inf, 1.0, inf, nan, -inf, inf], [-inf, inf, 3.0, 4.0, 5.0, 6.0]]
    x = torch.full((100, vocab), -inf)
    for r in range(100):
        at = torch.randperm(vocab, generator=g)
        x[r, at[:6]] = torch.tensor(heads[r % 5])
        if r % 2:
            x[r, at[6:vocab // 2]] = torch.randn(vocab // 2 - 6, generator=g) * 3
    x = x.to(dtype)
    check(cuda, x, torch.rand(100, generator=g), settings(100, g, "tkpm"))
    x = (torch.randn(24, vocab, generator=g) * 3).to(dtype)
    x[:, 5] = -inf
    t = torch.tensor([0.0, 1e-45, 1e-30, 1e-6, 1e-3, 1e3, 1e30, inf, 0.0, 2.0, inf, 1.0]).repeat(2)
    for which in ("", "kpm"):
        check(cuda, x, torch.rand(24, generator=g), dict(settings(24, g, which), temperature=t))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(300, 65400), (300, 65528), (150, 130900), (300, 131000), (8, 65528)])
def test_rows_of_one_bin(cuda, rows, vocab, dtype):
    """A few largest logits and all others equal: nearly the whole of a CTA's stretch falls into
    one bin of top-p's histogram, in the half of it whose weights are above its middle's, at
    stretches just below a power of two. The bulk's places in the histogram are in bins of
    their own order, from the first few to the last that has much weight."""
    bits = min(51, 62 - math.ceil(math.log2(vocab)))
    per_logit = 1.4426950408889634 * 4094.5 / (bits + 2)
    gaps = torch.linspace(0.02, 12.0, 6000).to(dtype).float().unique()
    part = (gaps.double() * per_logit) % 1
    gaps = gaps[(part > 0.505) & (part < 0.56)]
    gaps = gaps[torch.linspace(0, len(gaps) - 1, 5).long()]
    x, p, u = [], [], []
    for gap in gaps.tolist():
        top = max(1, round(vocab * math.exp(-gap) / 3))  # the bulk has about three quarters of the row
        row = torch.full((vocab,), 2.0 - gap).to(dtype)
        row[torch.randperm(vocab, generator=gen(top))[:top]] = 2.0
        below = 2.0 - float(row.float().min())  # after its rounding
        share = top / (top + (vocab - top) * math.exp(-below))
        for at in (0.6 * share, share + 0.3 * (1 - share), share + 0.8 * (1 - share)):
            x.append(row)
            p.append(at)
            u.append(0.9)
    n = len(x)
    x, p, u = torch.stack(x), torch.tensor(p), torch.tensor(u)
    none = dict(temperature=None, top_k=None, min_p=None)
    want = torch.tensor(ref.sample(x, u, top_p=p, **none), dtype=torch.int32)
    pick = torch.arange(rows) % n
    got = ops.sample(x.to(cuda)[pick.to(cuda)], u[pick].to(cuda), top_p=p[pick].to(cuda)).cpu()
    assert torch.equal(got, want[pick])
