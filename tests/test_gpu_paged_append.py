"""The paged append on the GPU: rotated K and V in their slots and nowhere else."""
import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, ops
from tests import serving_ref as ref
from tests.helpers import bits_equal, gen, randn

pytestmark = pytest.mark.gpu


def paged(cuda, g, num_pages, hkv, page, hd, dtype, table):
    k, v = (randn((num_pages, hkv, page, hd), dtype, g).to(cuda) for _ in range(2))
    return ops.PagedKV(k, v, torch.tensor(table, dtype=torch.int32, device=cuda))


def i32(values, cuda):
    return torch.tensor(values, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,hd,rd,page", [(32, 8, 128, 128, 16), (6, 6, 48, 24, 24), (2, 1, 64, 64, 1), (7, 1, 256, 64, 100),
                                               (3, 3, 6, 4, 5), (4, 2, 80, 80, 8)])
@pytest.mark.parametrize("rows", [1, 37, 2100])
def test_append(cuda, rows, hq, hkv, hd, rd, page, interleaved, dtype):
    g = gen(rows + hd)
    num_seqs = 3
    per = -(-rows // num_seqs)
    max_pages = -(-(per + 11) // page) + 1
    ids = torch.randperm(num_seqs * max_pages, generator=g).view(num_seqs, max_pages).tolist()
    cache = paged(cuda, g, num_seqs * max_pages, hkv, page, hd, dtype, ids)
    q, k, v = randn((rows, hq, hd), dtype, g), randn((rows, hkv, hd), dtype, g), randn((rows, hkv, hd), dtype, g)
    seqs = [r % num_seqs for r in range(rows)]
    slots = [11 + r // num_seqs for r in range(rows)]
    pos = torch.randint(0, 3000, (rows,), generator=g, dtype=torch.int32)
    table, st = ops.RopeTable(3000, rd, 1e4, cuda), ops.DeviceStatus(cuda)
    k_before, v_before = cache.k_pages.clone(), cache.v_pages.clone()
    qo = ops.paged_kv_append(q.to(cuda), k.to(cuda), v.to(cuda), pos.to(cuda), cache, table=table, seq_ids=i32(seqs, cuda),
                             slots=i32(slots, cuda), interleaved=interleaved, status=st)
    assert st.read() == 0
    rq, rk = ops.rotary(q.to(cuda), k.to(cuda), pos.to(cuda), table, interleaved=interleaved)
    assert bits_equal(qo, rq)
    f = ref.frequencies(rd, 1e4)
    want, pair = ref.rotated(k, pos.numpy(), f, 1.0, interleaved)
    assert np.all(np.abs(rk.cpu().double().numpy() - want) <= ref.rotation_tolerance(want, pair, 1.0, dtype))
    page_of = torch.tensor([ids[s][t // page] for s, t in zip(seqs, slots)], device=cuda)
    off = torch.tensor([t % page for t in slots], device=cuda)
    k_before[page_of, :, off] = rk
    v_before[page_of, :, off] = v.to(cuda)
    assert bits_equal(cache.k_pages, k_before) and bits_equal(cache.v_pages, v_before)


def test_slots_are_positions_and_no_rotation(cuda):
    g = gen(5)
    cache = paged(cuda, g, 4, 2, 8, 32, torch.bfloat16, [[2, 0], [3, 1]])
    q, k, v = (randn((3, h, 32), torch.bfloat16, g).to(cuda) for h in (4, 2, 2))
    pos = i32([9, 0, 7], cuda)
    seq = i32([0, 1, 1], cuda)
    qo = ops.paged_kv_append(q, k, v, pos, cache, seq_ids=seq)
    assert bits_equal(qo, q)
    for r, (page, off) in enumerate([(0, 1), (3, 0), (3, 7)]):
        assert bits_equal(cache.k_pages[page, :, off], k[r]) and bits_equal(cache.v_pages[page, :, off], v[r])
    assert ops.paged_kv_append(None, k, v, None, cache, slots=pos, seq_ids=seq) is None  # no q, no positions
    table = ops.RopeTable(32, 32, 1e4, cuda)
    same = q.clone()
    out = ops.paged_kv_append(same, k, v, pos, cache, table=table, seq_ids=seq, q_out=same)  # in place
    assert out is same and bits_equal(same, ops.rotary(q, None, pos, table)[0])


def test_padding_and_bad_rows_are_skipped(cuda):
    g = gen(6)
    cache = paged(cuda, g, 4, 1, 8, 32, torch.float32, [[2, 0], [9, -3]])
    before = cache.k_pages.clone(), cache.v_pages.clone()
    q, k, v = (randn((9, h, 32), torch.float32, g).to(cuda) for h in (2, 1, 1))
    table, st = ops.RopeTable(20, 32, 1e4, cuda), ops.DeviceStatus(cuda)
    qo = torch.full_like(q, 3.0)

    def go(pos, slots, seqs):
        ops.paged_kv_append(q[:len(pos)], k[:len(pos)], v[:len(pos)], i32(pos, cuda), cache, table=table,
                            seq_ids=i32(seqs, cuda), slots=None if slots is None else i32(slots, cuda),
                            q_out=qo[:len(pos)], status=st)
        return st.read()

    assert go([-1, -7, 25], [-1, -1, -1], [0, 99, -4]) == 0        # padding, whatever else the row says
    assert go([-1], None, [0]) == 0
    assert go([20], [0], [0]) == _lib.BM_DEVERR_BAD_POSITION         # past the table
    assert go([-2], None, [0]) == _lib.BM_DEVERR_BAD_POSITION
    assert go([3], [16], [0]) == _lib.BM_DEVERR_BAD_POSITION         # past max_pages
    assert go([3], [-2], [0]) == _lib.BM_DEVERR_BAD_POSITION
    assert go([3], [3], [2]) == _lib.BM_DEVERR_BAD_SEQUENCE
    assert go([3], [3], [-1]) == _lib.BM_DEVERR_BAD_SEQUENCE
    assert go([3, 3], [3, 8], [1, 1]) == _lib.BM_DEVERR_BAD_PAGE     # pages 9 and -3 of 4
    assert bits_equal(qo, torch.full_like(q, 3.0))
    assert bits_equal(cache.k_pages, before[0]) and bits_equal(cache.v_pages, before[1])
    assert go([20, 5], [0, 5], [0, 0]) == _lib.BM_DEVERR_BAD_POSITION  # a good row beside a bad one
    assert bits_equal(cache.v_pages[2, :, 5], v[1])


def test_slices_of_a_fused_projection(cuda):
    g = gen(7)
    cache = paged(cuda, g, 6, 2, 16, 64, torch.bfloat16, [[1, 4, 5]])
    qkv = randn((33, 8, 64), torch.bfloat16, g).to(cuda)
    pos = torch.arange(33, dtype=torch.int32, device=cuda)
    table = ops.RopeTable(40, 64, 1e4, cuda)
    want = ops.paged_kv_append(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), qkv[:, 6:].contiguous(), pos, cache,
                               table=table)
    kept = cache.k_pages.clone(), cache.v_pages.clone()
    cache.k_pages[[1, 4, 5]] = 0
    cache.v_pages[[1, 4, 5]] = 0
    got = ops.paged_kv_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], pos, cache, table=table, q_out=qkv[:, :4])
    assert bits_equal(got, want)
    assert bits_equal(cache.k_pages[[1, 4]], kept[0][[1, 4]]) and bits_equal(cache.v_pages[[1, 4]], kept[1][[1, 4]])
    assert bits_equal(cache.k_pages[5, :, 0], kept[0][5, :, 0])


def test_pages_past_32_bit_offsets(cuda):
    """A cache of over 2^31 elements: the last page's slots land where they belong."""
    hkv, page, hd = 8, 256, 128
    num_pages = 2 ** 31 // (hkv * page * hd) + 2
    k = torch.zeros(num_pages, hkv, page, hd, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros_like(k)
    cache = ops.PagedKV(k, v, torch.tensor([[num_pages - 1, 0]], dtype=torch.int32, device=cuda))
    x = randn((1, hkv, hd), torch.bfloat16, gen(8)).to(cuda)
    ops.paged_kv_append(None, x, x, i32([255], cuda), cache)
    assert bits_equal(k[-1, :, 255], x[0]) and bits_equal(v[-1, :, 255], x[0])
    assert int(torch.count_nonzero(k[0])) == 0
    out = ops.paged_tree_attention(torch.ones(1, 8, hd, dtype=torch.bfloat16, device=cuda), cache, i32([255], cuda),
                                   i32([0, 1], cuda), 255, 1)
    assert bool(torch.isfinite(out).all()) and int(torch.count_nonzero(out)) > 0


def test_another_stream_and_a_captured_graph(cuda):
    g = gen(9)
    cache = paged(cuda, g, 6, 2, 16, 64, torch.bfloat16, [[1, 4, 5]])
    q, k, v = (randn((5, h, 64), torch.bfloat16, g).to(cuda) for h in (4, 2, 2))
    pos = i32([0, 1, 2, 30, 31], cuda)
    table = ops.RopeTable(40, 64, 1e4, cuda)
    want = ops.paged_kv_append(q, k, v, pos, cache, table=table)
    kept = cache.k_pages.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.paged_kv_append(q, k, v, pos, cache, table=table, stream=side)
    side.synchronize()
    assert bits_equal(got, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(q, k, v, pos, cache, table=table, q_out=out)
    cache.k_pages[[1, 4, 5]] = 0
    pos.copy_(i32([3, 1, 2, 30, 31], cuda))
    graph.replay()
    torch.cuda.synchronize()
    assert bits_equal(cache.k_pages[1, :, 1], kept[1, :, 1]) and int(torch.count_nonzero(cache.k_pages[1, :, 3])) > 0
    assert int(torch.count_nonzero(cache.k_pages[1, :, 0])) == 0 and bits_equal(out[1:], want[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_cache_whose_tensors_are_replaced(cuda, dtype):
    """Calls go by the tensors that a PagedKV holds at the time: other pages, other page tables,
    more of either; what no longer fits together is refused."""
    g = gen(10)
    cache = paged(cuda, g, 4, 2, 8, 64, dtype, [[2, 0], [3, 1]])
    old = cache.k_pages, cache.v_pages, cache.page_table
    kept = [t.clone() for t in old]
    q, k, v = (randn((3, h, 64), dtype, g).to(cuda) for h in (4, 2, 2))
    pos, ones = i32([0, 1, 2], cuda), i32([1, 1, 1], cuda)
    new = paged(cuda, g, 7, 2, 8, 64, dtype, [[0, 1, 2], [6, 5, 4]])
    want = paged(cuda, g, 7, 2, 8, 64, dtype, [[0, 1, 2], [6, 5, 4]])
    want.k_pages.copy_(new.k_pages)
    want.v_pages.copy_(new.v_pages)
    ops.paged_kv_append(None, k, v, pos, want, seq_ids=ones)
    cache.k_pages, cache.v_pages, cache.page_table = new.k_pages, new.v_pages, new.page_table
    assert (cache.num_pages, cache.num_seqs, cache.max_pages) == (7, 2, 3)
    ops.paged_kv_append(None, k, v, pos, cache, seq_ids=ones)
    assert bits_equal(cache.k_pages, want.k_pages) and bits_equal(cache.v_pages, want.v_pages)
    for t, was in zip(old, kept):
        assert bits_equal(t, was)
    args = i32([0], cuda), i32([0, 3], cuda), 0, 3
    ids = i32([1], cuda)
    assert bits_equal(ops.paged_tree_attention(q, cache, *args, seq_ids=ids),
                      ops.paged_tree_attention(q, want, *args, seq_ids=ids))
    for name, bad in (("k_pages", new.k_pages[:6]), ("v_pages", new.v_pages.to(torch.float64)),
                      ("v_pages", new.v_pages.transpose(0, 1)), ("k_pages", new.k_pages.cpu()), ("page_table", new.page_table.long()),
                      ("page_table", new.page_table[:, :2]), ("page_table", new.page_table[0]), ("page_table", None)):
        good = getattr(cache, name)
        setattr(cache, name, bad)
        with pytest.raises(_lib.BMError):
            ops.paged_kv_append(None, k, v, pos, cache, seq_ids=ones)
        with pytest.raises(_lib.BMError):
            ops.paged_tree_attention(q, cache, *args, seq_ids=ids, workspace=torch.empty(1 << 20, dtype=torch.uint8, device=cuda))
        setattr(cache, name, good)
    assert bits_equal(cache.k_pages, want.k_pages) and bits_equal(cache.v_pages, want.v_pages)
