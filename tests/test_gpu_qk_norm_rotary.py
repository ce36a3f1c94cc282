"""Norms of Q's and K's heads with their rotation in one pass, on the GPU against 64 bits."""
import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import kv8_ref, serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
THETA = 1e4


def check(got, x, w, eps, positions, rd, interleaved, dtype, rows=None):
    want, off = kv8_ref.turned(x, w, eps, positions, ref.frequencies(rd, THETA), interleaved)
    tol = off + ref.HALF[dtype] * (np.abs(want) + off) * 1.01
    err = np.abs(got.cpu().double().numpy() - want)
    keep = slice(None) if rows is None else rows
    assert np.all(err[keep] <= tol[keep]), np.max((err - tol)[keep])


def heads(rows, hq, hkv, hd, dtype, seed=0):
    g = gen(seed)
    qkv = randn((rows, hq + 2 * hkv, hd), dtype, g, scale=3.0)
    return qkv, randn((hd,), dtype, g, scale=0.3, offset=1.0), randn((hd,), dtype, g, scale=0.3, offset=1.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,hq,hkv,hd,rd", [
    (1, 1, 1, 128, 128), (64, 32, 8, 128, 128), (3, 7, 1, 128, 64), (130, 6, 6, 48, 48), (5, 6, 6, 48, 24), (2, 4, 2, 256, 256),
    (9, 3, 2, 64, 16), (4, 5, 1, 80, 80), (7, 2, 2, 10, 6), (3, 3, 1, 33, 32), (2, 2, 1, 255, 2), (6, 1, 1, 2, 2),
    (2100, 2, 1, 96, 32), (3, 9, 4, 250, 120), (4, 3, 1, 112, 24)])
def test_against_64_bits(cuda, dtype, interleaved, rows, hq, hkv, hd, rd):
    """q and k are slices of a fused projection's rows; the outputs are dense."""
    qkv, wq, wk = heads(rows, hq, hkv, hd, dtype, seed=rows + hd)
    table = ops.RopeTable(700, rd, THETA, cuda)
    pos = torch.randint(0, 700, (rows,), generator=gen(1), dtype=torch.int32)
    d, st = qkv.to(cuda), ops.DeviceStatus(cuda)
    q, k = ops.qk_norm_rotary(d[:, :hq], d[:, hq:hq + hkv], wq.to(cuda), wk.to(cuda), pos.to(cuda), table, eps=1e-4,
                              interleaved=interleaved, status=st)
    assert st.read() == 0
    check(q, qkv[:, :hq], wq, 1e-4, pos.numpy(), rd, interleaved, dtype)
    check(k, qkv[:, hq:hq + hkv], wk, 1e-4, pos.numpy(), rd, interleaved, dtype)
    assert bits_equal(d, qkv)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_of_the_two_in_place_and_from_a_position_on(cuda, dtype):
    qkv, wq, wk = heads(20, 4, 2, 64, dtype)
    table = ops.RopeTable(64, 64, THETA, cuda)
    both = ops.qk_norm_rotary(qkv[:, :4].to(cuda), qkv[:, 4:6].to(cuda), wq.to(cuda), wk.to(cuda), 7, table)
    d = qkv.to(cuda)
    q, none = ops.qk_norm_rotary(d[:, :4], None, wq.to(cuda), None, 7, table, q_out=d[:, :4])
    none2, k = ops.qk_norm_rotary(None, d[:, 4:6], None, wk.to(cuda), 7, table, k_out=d[:, 4:6])
    assert none is None and none2 is None
    assert bits_equal(q, both[0]) and bits_equal(k, both[1]) and bits_equal(d[:, :4], both[0])
    assert bits_equal(d[:, 6:], qkv[:, 6:])
    check(both[0], qkv[:, :4], wq, 1e-5, np.arange(7, 27), 64, False, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rows_off_16_byte_boundaries(cuda, dtype, shift):
    """Narrower chunks and single elements give the same values up to the sum's order."""
    rows, hq, hd = 5, 3, 128
    qkv, wq, _ = heads(rows, hq, 1, hd, dtype, seed=3)
    wide = torch.zeros(rows, hq * hd + 8, dtype=dtype, device=cuda)
    view = torch.as_strided(wide, (rows, hq, hd), (hq * hd + 8, hd, 1), shift)
    view.copy_(qkv[:, :hq])
    table = ops.RopeTable(64, hd, THETA, cuda)
    q, _ = ops.qk_norm_rotary(view, None, wq.to(cuda), None, 3, table)
    check(q, qkv[:, :hq], wq, 1e-5, np.arange(3, 3 + rows), hd, False, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_zeros_and_values_that_are_not_finite(cuda, dtype):
    qkv, wq, _ = heads(4, 3, 1, 64, dtype)
    q = qkv[:, :3].clone()
    q[0, 0] = 0.0
    q[1, 1, 5] = float("inf")
    q[2, 2, 6] = float("nan")
    table = ops.RopeTable(64, 64, THETA, cuda)
    got, _ = ops.qk_norm_rotary(q.to(cuda), None, wq.to(cuda), None, 0, table)
    got = got.cpu()
    assert torch.count_nonzero(got[0, 0]) == 0
    assert torch.isnan(got[1, 1]).any() and torch.isnan(got[2, 2]).all()
    clean = torch.ones(4, 3, dtype=torch.bool)
    clean[1, 1] = clean[2, 2] = False
    assert torch.isfinite(got[clean]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_positions_are_flagged_and_their_rows_left(cuda, dtype):
    qkv, wq, wk = heads(6, 2, 1, 64, dtype)
    table = ops.RopeTable(10, 64, THETA, cuda)
    pos = torch.tensor([3, -1, 9, 10, 0, 2 ** 31 - 1], dtype=torch.int32)
    qo, ko = torch.full((6, 2, 64), 5.0, dtype=dtype, device=cuda), torch.full((6, 1, 64), 5.0, dtype=dtype, device=cuda)
    st = ops.DeviceStatus(cuda)
    ops.qk_norm_rotary(qkv[:, :2].to(cuda), qkv[:, 2:3].to(cuda), wq.to(cuda), wk.to(cuda), pos.to(cuda), table, q_out=qo,
                       k_out=ko, status=st)
    assert st.read() == _lib.BM_DEVERR_BAD_POSITION
    check(qo, qkv[:, :2], wq, 1e-5, pos.clamp(0, 9).numpy(), 64, False, dtype, rows=[0, 2, 4])
    for r in (1, 3, 5):
        assert bool((qo[r] == 5.0).all()) and bool((ko[r] == 5.0).all())


def test_streams_and_graphs(cuda):
    qkv, wq, wk = heads(70, 8, 2, 128, BF16)
    d, wq, wk = qkv.to(cuda), wq.to(cuda), wk.to(cuda)
    table = ops.RopeTable(128, 128, THETA, cuda)
    args = (d[:, :8], d[:, 8:10], wq, wk, 1, table)
    first = ops.qk_norm_rotary(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = ops.qk_norm_rotary(*args, stream=side)
    side.synchronize()
    assert all(bits_equal(a, b) for a, b in zip(first, other))
    outs = [torch.empty_like(t) for t in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.qk_norm_rotary(*args, q_out=outs[0], k_out=outs[1])
    for _ in range(2):
        for t in outs:
            t.zero_()
        graph.replay()
        assert all(bits_equal(a, b) for a, b in zip(first, outs))


def test_no_rows(cuda):
    table = ops.RopeTable(8, 64, THETA, cuda)
    w = torch.ones(64, dtype=BF16, device=cuda)
    q, k = ops.qk_norm_rotary(torch.empty(0, 4, 64, dtype=BF16, device=cuda), None, w, None, 0, table)
    assert q.shape == (0, 4, 64) and k is None
