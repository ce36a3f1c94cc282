"""Rotary forms on the GPU against 64-bit rotations: pairings, part of the head, scaled
tables, slices of wider rows, in place, bad positions."""
import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

SCALINGS = {
    "none": (None, {}),
    "linear": (ops.RopeScaling("linear", 4.0), dict(kind="linear", factor=4.0)),
    "ntk": (ops.RopeScaling("ntk", 8.0), dict(kind="ntk", factor=8.0)),
    "bands": (ops.RopeScaling("bands", 8.0, 512, low_freq_factor=1.0, high_freq_factor=4.0),
              dict(kind="bands", factor=8.0, original_max_pos=512, low=1.0, high=4.0)),
    "yarn": (ops.RopeScaling("yarn", 16.0, 512, beta_fast=32.0, beta_slow=1.0),
             dict(kind="yarn", factor=16.0, original_max_pos=512, low=32.0, high=1.0)),
}


def mscale(name):
    return 0.1 * np.log(16.0) + 1.0 if name == "yarn" else 1.0


@pytest.mark.parametrize("name", SCALINGS)
@pytest.mark.parametrize("dim,theta,max_pos", [(128, 5e5, 4097), (24, 1e4, 1000), (4, 1e4, 3)])
def test_tables(cuda, name, dim, theta, max_pos):
    t = ops.RopeTable(max_pos, dim, theta, cuda, scaling=SCALINGS[name][0])
    f = ref.frequencies(dim, theta, **SCALINGS[name][1])
    angle = np.arange(max_pos)[:, None] * f[None]
    want = mscale(name) * np.stack([np.cos(angle), np.sin(angle)], -1)
    got = t.data.cpu().double().numpy()
    # one rounding to fp32 of a 64-bit value (angles up to 4097: 2^12 * 2^-52 * a few)
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -36)


def test_table_of_no_scaling_is_the_rope_table(cuda):
    a = ops.RopeTable(300, 64, 1e4, cuda)
    assert bits_equal(a.data, ops.RopeTable(300, 64, 1e4, cuda, scaling=ops.RopeScaling()).data)
    assert not bits_equal(a.data, ops.RopeTable(300, 64, 1e4, cuda, scaling=ops.RopeScaling(mscale=0.5)).data)


def check(cuda, rows, hq, hkv, hd, rd, interleaved, dtype, scaling="none", max_pos=700, seed=0):
    g = gen(seed)
    q, k = randn((rows, hq, hd), dtype, g), randn((rows, hkv, hd), dtype, g)
    pos = torch.randint(0, max_pos, (rows,), generator=g, dtype=torch.int32)
    table = ops.RopeTable(max_pos, rd, 1e4, cuda, scaling=SCALINGS[scaling][0])
    f = ref.frequencies(rd, 1e4, **SCALINGS[scaling][1])
    st = ops.DeviceStatus(cuda)
    qd, kd = q.to(cuda), k.to(cuda)
    got = ops.rotary(qd, kd, pos.to(cuda), table, interleaved=interleaved, status=st)
    assert st.read() == 0
    for x, dev, o in ((q, qd, got[0]), (k, kd, got[1])):
        want, pair = ref.rotated(x, pos.numpy(), f, mscale(scaling), interleaved)
        err = np.abs(o.cpu().double().numpy() - want)
        assert np.all(err <= ref.rotation_tolerance(want, pair, mscale(scaling), dtype)), err.max()
        assert bits_equal(dev, x)  # the input is left alone
    return q, k, pos, table, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hkv,hd,rd", [
    (1, 32, 8, 128, 128), (64, 32, 8, 128, 128), (3, 1, 1, 2, 2), (5, 3, 1, 6, 4), (7, 6, 6, 48, 48), (7, 6, 6, 48, 24),
    (9, 4, 2, 256, 64), (2, 2, 1, 1024, 1024), (3, 2, 2, 520, 514), (2500, 4, 1, 64, 32), (2500, 3, 1, 80, 40)])
def test_rotary(cuda, rows, hq, hkv, hd, rd, interleaved, dtype):
    check(cuda, rows, hq, hkv, hd, rd, interleaved, dtype)


@pytest.mark.parametrize("name", list(SCALINGS)[1:])
def test_scaled(cuda, name):
    check(cuda, 33, 4, 2, 64, 64, True, torch.bfloat16, scaling=name, max_pos=5000)


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equals_rope_bit_for_bit(cuda, rows, dtype):
    q, k, pos, table, got = check(cuda, rows, 4, 2, 128, 128, False, dtype)
    qd, kd = q.to(cuda), k.to(cuda)
    ops.rope(qd, kd, pos.to(cuda), table)
    assert bits_equal(qd, got[0]) and bits_equal(kd, got[1])


@pytest.mark.parametrize("rd", [64, 24])
def test_slices_in_place_and_one_tensor(cuda, rd):
    """q and k inside a fused projection's rows, rotated where they stand: v, and elements
    past each row's heads, keep their bits; an odd offset takes the scalar path."""
    g, table = gen(1), ops.RopeTable(50, rd, 1e4, cuda)
    for lead in (0, 1):
        base = randn((17, lead + 8 * 64 + 5), torch.bfloat16, g).to(cuda)
        before = base.clone()
        qkv = base[:, lead:lead + 8 * 64].unflatten(1, (8, 64))
        pos = torch.randint(0, 50, (17,), generator=g, dtype=torch.int32).to(cuda)
        apart = ops.rotary(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), pos, table)
        ops.rotary(qkv[:, :4], qkv[:, 4:6], pos, table, q_out=qkv[:, :4], k_out=qkv[:, 4:6])
        assert bits_equal(qkv[:, :4], apart[0]) and bits_equal(qkv[:, 4:6], apart[1])
        rest = torch.ones_like(base, dtype=torch.bool)
        rest[:, lead:lead + 6 * 64] = False
        assert bits_equal(base[rest], before[rest])
        only, none = ops.rotary(before[:, lead:lead + 256].unflatten(1, (4, 64)), None, pos, table)
        assert none is None and bits_equal(only, apart[0])


def test_bad_positions_leave_their_rows(cuda):
    g = gen(2)
    q, k = randn((6, 2, 32), torch.float32, g).to(cuda), randn((6, 1, 32), torch.float32, g).to(cuda)
    table, st = ops.RopeTable(10, 32, 1e4, cuda), ops.DeviceStatus(cuda)
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    ops.rotary(q, k, torch.tensor([0, 10, 9, -1, 2, 2 ** 30], dtype=torch.int32, device=cuda), table, q_out=qo, k_out=ko,
               status=st)
    assert st.read() == _lib.BM_DEVERR_BAD_POSITION
    good = ops.rotary(q, k, torch.tensor([0, 0, 9, 0, 2, 0], dtype=torch.int32, device=cuda), table)
    for o, w in ((qo, good[0]), (ko, good[1])):
        for r in range(6):
            assert bits_equal(o[r], w[r] if r in (0, 2, 4) else torch.full_like(w[r], 7.0))
    a = ops.rotary(q, k, 4, table)  # pos0: rows 4..9
    b = ops.rotary(q, k, torch.arange(4, 10, dtype=torch.int32, device=cuda), table)
    assert bits_equal(a[0], b[0]) and bits_equal(a[1], b[1])


def test_no_rows(cuda):
    table = ops.RopeTable(10, 32, 1e4, cuda)
    z = torch.empty(0, 2, 32, device=cuda)
    assert ops.rotary(z, None, torch.empty(0, dtype=torch.int32, device=cuda), table)[0].shape == (0, 2, 32)


def test_a_table_smaller_than_it_says_is_refused(cuda):
    """A table's tensor and its sizes go into a call apart: kernels would read past the
    tensor where the sizes say more. (Refused on the host; nothing is launched.)"""
    q = randn((3, 2, 32), torch.float32, gen(3)).to(cuda)
    pos = torch.zeros(3, dtype=torch.int32, device=cuda)
    pages = torch.zeros(1, 2, 8, 32, device=cuda)
    cache = ops.PagedKV(pages, pages.clone(), torch.zeros(1, 1, dtype=torch.int32, device=cuda))
    for name, value in (("data", torch.zeros(9, 12, 2, device=cuda)), ("data", torch.zeros(10, 12, 2, dtype=torch.float64, device=cuda)),
                        ("data", torch.zeros(10, 2, 12, device=cuda).transpose(1, 2)), ("max_pos", 11), ("head_dim", 26)):
        table = ops.RopeTable(10, 24, 1e4, cuda)
        setattr(table, name, value)
        with pytest.raises(_lib.BMError):
            ops.rotary(q, None, pos, table)
        with pytest.raises(_lib.BMError):
            ops.paged_kv_append(None, q, q, pos, cache, table=table)
    assert int(torch.count_nonzero(pages)) == 0
