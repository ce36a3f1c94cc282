"""CPU-side refusals of the 8-bit paged cache's entry points and of qk_norm_rotary: bad arguments
are rejected on the host before anything reaches CUDA, empty calls do nothing, and the struct
mirrors the header's."""
import ctypes

import numpy as np
import pytest
import torch

from baremetalinferenceengine_b200 import _lib, build, ops
from tests import kv8_ref
from tests.test_serving_refusals import test_struct_layouts_match_the_header as same_layout

FAKE = 0x1000000  # never dereferenced: every call below fails or returns before any CUDA call
FAR = 0x4000000
W = 0x8000000


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def cache(**kw):
    c = dict(k_pages=W * 2, v_pages=W * 3, k_scales=W * 4, v_scales=W * 5, page_table=W * 6, num_pages=4, page_size=8, block=4,
             max_pages=2, num_seqs=2, num_kv_heads=2, head_dim=64)
    c.update(kw)
    return ctypes.byref(_lib.PagedKV8C(*[c[n] for n, _ in _lib.PagedKV8C._fields_]))


def norm(L, qo=FAR, ko=FAR * 2, q=FAKE, k=FAKE * 2, wq=W, wk=W + 4096, eps=1e-5, pos=FAKE, pos0=0, table=FAKE, n=8, rd=64, rows=4,
         hq=4, hkv=2, hd=64, qs=256, ks=128, qos=256, kos=128, dtype=0, status=None):
    return L.bm_qk_norm_rotary(qo, ko, q, k, wq, wk, eps, pos, pos0, table, n, rd, 0, rows, hq, hkv, hd, qs, ks, qos, kos, dtype,
                               status, None)


def append(L, qo=FAR, q=FAKE, k=FAKE * 2, v=FAKE * 3, wq=W, wk=W + 4096, eps=1e-5, pos=FAKE, c=None, seqs=None, ctx=FAKE, starts=FAKE,
           table=FAKE, n=8, rd=64, rows=4, batch=2, hq=4, most=4, qs=256, ks=128, vs=128, qos=256, dtype=0, status=None):
    return L.bm_paged_kv8_append(qo, q, k, v, wq, wk, eps, pos, c or cache(), seqs, ctx, starts, table, n, rd, 0, rows, batch, hq, most,
                                 qs, ks, vs, qos, dtype, status, None)


def read(L, ko=FAR, vo=FAR * 2, c=None, seqs=None, first=FAKE, starts=FAKE, rows=4, batch=2, most=4, dtype=0, status=None):
    return L.bm_paged_kv8_read(ko, vo, c or cache(), seqs, first, starts, rows, batch, most, dtype, status, None)


def attend(L, out=FAR, q=FAKE, c=None, ctx=FAKE, starts=FAKE, mask=FAKE, words=1, total=4, batch=2, hq=4, max_ctx=8,
           max_tree=4, scale=0.0, ws=FAR * 4, ws_bytes=1 << 40, dtype=0, seqs=None, status=None):
    return L.bm_paged_kv8_tree_attention(out, q, c or cache(), seqs, ctx, starts, mask, words, total, batch, hq, max_ctx,
                                         max_tree, scale, ws, ws_bytes, dtype, status, None)


def size(L, total=4, batch=2, hq=4, hkv=2, hd=64, max_ctx=8, max_tree=4, out=True):
    return L.bm_paged_kv8_tree_attention_workspace_size(total, batch, hq, hkv, hd, max_ctx, max_tree,
                                                        ctypes.byref(ctypes.c_size_t()) if out else None)


BAD_CACHES = [dict(k_pages=None), dict(v_pages=None), dict(k_scales=None), dict(v_scales=None), dict(page_table=None), dict(num_pages=0),
              dict(page_size=0), dict(block=0), dict(block=-4), dict(block=3), dict(block=16), dict(max_pages=-1), dict(num_seqs=0),
              dict(num_kv_heads=0), dict(num_kv_heads=(1 << 16) + 1), dict(head_dim=0), dict(head_dim=8), dict(head_dim=72),
              dict(head_dim=272), dict(page_size=1 << 20, max_pages=1 << 12), dict(page_size=8, block=8, max_pages=(1 << 28) - 1), dict(k_pages=W * 2 + 8), dict(v_pages=W * 3 + 4),
              dict(page_table=W * 6 + 2)]


@pytest.mark.parametrize("bad", BAD_CACHES)
@pytest.mark.parametrize("call", [append, read, attend])
def test_bad_caches(lib, call, bad):
    assert call(lib, c=cache(**bad)) == _lib.BM_ERR_INVALID_ARGUMENT
    assert lib.bm_last_error_message()


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("call,kw", [(norm, k) for k in [
    dict(dtype=3), dict(rows=-1), dict(rows=1 << 31), dict(hq=-1), dict(hkv=(1 << 16) + 1), dict(hd=0), dict(hd=257), dict(eps=-1.0),
    dict(eps=NAN), dict(eps=INF), dict(table=None), dict(n=0), dict(table=FAKE + 4), dict(rd=7), dict(rd=0), dict(rd=66), dict(q=None),
    dict(ko=None), dict(wq=None), dict(wk=None), dict(qs=255), dict(kos=64), dict(pos=None, pos0=-1), dict(pos=None, pos0=2 ** 31 - 3),
    dict(qo=FAKE + 4), dict(qo=FAKE, qos=300), dict(qo=FAKE * 2), dict(ko=FAR + 16), dict(qo=W - 64), dict(ko=W + 4096 + 252),
    dict(qo=W + 4096), dict(q=FAKE + 2), dict(k=FAKE * 2 + 1), dict(wq=W + 2), dict(wk=W + 1, dtype=1), dict(qo=FAR + 1, dtype=1),
    dict(pos=FAKE + 2), dict(status=FAKE + 2)]] + [(append, k) for k in [
        dict(dtype=2), dict(rows=-2), dict(batch=-1), dict(most=-1), dict(hq=-1), dict(eps=NAN), dict(eps=-1e-5), dict(k=None),
        dict(v=None), dict(q=None), dict(qo=None), dict(ctx=None), dict(starts=None), dict(n=0), dict(rd=65), dict(rd=128), dict(ks=127),
        dict(vs=0), dict(qos=1), dict(batch=3), dict(qo=FAKE + 16), dict(qo=FAKE * 3), dict(qo=W - 64), dict(qo=W + 4096),
        dict(qo=W * 2), dict(qo=W * 3 + 4092), dict(qo=W * 4), dict(k=W * 2 - 4), dict(v=W * 5), dict(q=W * 3), dict(q=FAKE + 2),
        dict(k=FAKE * 2 + 2), dict(v=FAKE * 3 + 1, dtype=1), dict(wq=W + 2), dict(wk=W + 1, dtype=1), dict(pos=FAKE + 1),
        dict(seqs=FAKE + 2), dict(ctx=FAKE + 2), dict(starts=FAKE + 3), dict(status=FAKE + 1),
        dict(most=2 ** 31 - 1, seqs=FAKE, batch=2 ** 31 - 1)]] + [(read, k) for k in [
            dict(dtype=5), dict(rows=-1), dict(batch=-1), dict(most=-1), dict(ko=None), dict(vo=None), dict(first=None), dict(starts=None),
            dict(batch=3), dict(ko=FAR + 8), dict(vo=FAR * 2 + 4), dict(vo=FAR + 16), dict(ko=W * 2), dict(vo=W * 3 + 4080), dict(ko=W * 5 - 16),
            dict(first=FAKE + 2), dict(starts=FAKE + 1), dict(seqs=FAKE + 2), dict(status=FAKE + 3),
            dict(most=2 ** 31 - 1, seqs=FAKE, batch=2 ** 31 - 1)]] + [(attend, k) for k in [
                dict(dtype=9), dict(total=-1), dict(batch=-1), dict(hq=3), dict(hq=0), dict(hq=130), dict(max_ctx=-1), dict(max_tree=-1),
                dict(max_ctx=1 << 30), dict(words=0), dict(max_tree=65), dict(scale=NAN), dict(scale=INF), dict(scale=3.4e38),
                dict(out=None), dict(q=None), dict(ctx=None), dict(starts=None), dict(q=FAKE + 4), dict(out=FAR + 8), dict(ws=FAR + 4),
                dict(out=FAKE + 64), dict(batch=3), dict(ws=None, max_ctx=4096), dict(ws_bytes=64, max_ctx=4096), dict(out=W * 2),
                dict(out=W * 3 + 4080), dict(out=W * 4), dict(out=W * 5 - 16), dict(ctx=FAKE + 2), dict(starts=FAKE + 1),
                dict(mask=FAKE + 4), dict(seqs=FAKE + 2), dict(status=FAKE + 2)]] + [(size, k) for k in [
                    dict(out=False), dict(hd=0), dict(hq=5), dict(total=-1), dict(batch=1 << 20, max_tree=1 << 10)]])
def test_host_checks_reject_before_any_launch(lib, call, kw):
    assert call(lib, **kw) == _lib.BM_ERR_INVALID_ARGUMENT
    assert lib.bm_last_error_message()


@pytest.mark.parametrize("call,kw", [
    (norm, dict(rows=0)), (norm, dict(hq=0, hkv=0)), (append, dict(rows=0)), (append, dict(batch=0)), (append, dict(most=0)),
    (read, dict(rows=0)), (read, dict(batch=0)), (read, dict(most=0)), (attend, dict(batch=0)), (attend, dict(total=0)),
    (attend, dict(max_tree=0)), (size, dict(batch=0)), (size, dict(max_tree=0))])
def test_empty_calls_are_no_ops(lib, call, kw):
    assert call(lib, **kw) == _lib.BM_OK


def test_struct_layout_matches_the_header():
    same_layout(_lib.PagedKV8C, "bm_paged_kv8_t")


def tensors(**kw):
    t = dict(k_pages=torch.zeros(4, 2, 8, 64, dtype=torch.float8_e4m3fn), v_pages=torch.zeros(4, 2, 8, 64, dtype=torch.float8_e4m3fn),
             k_scales=torch.zeros(4, 2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu),
             v_scales=torch.zeros(4, 2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu), page_table=torch.zeros(2, 2, dtype=torch.int32))
    t.update(kw)
    return t


@pytest.mark.parametrize("kw,text", [
    (dict(), "CUDA"), (dict(k_pages=torch.zeros(4, 2, 8, 64)), "float8_e4m3fn"), (dict(k_pages=torch.zeros(2, 8, 64)), "num_pages"),
    (dict(v_pages=torch.zeros(4, 2, 4, 64, dtype=torch.float8_e4m3fn)), "num_pages"),
    (dict(k_scales=torch.zeros(4, 2, 2)), "e8m0"), (dict(k_scales=torch.zeros(4, 2, 3, dtype=torch.uint8).view(torch.float8_e8m0fnu),
                                                         v_scales=torch.zeros(4, 2, 3, dtype=torch.uint8).view(torch.float8_e8m0fnu)), "scales")])
def test_the_python_cache_refuses(kw, text):
    with pytest.raises(_lib.BMError, match=text):
        ops.PagedKV8(**tensors(**kw))


@pytest.mark.parametrize("hd", [8, 24, 272])
def test_the_python_cache_refuses_other_head_sizes(hd):
    pages = [torch.zeros(4, 2, 8, hd, dtype=torch.float8_e4m3fn) for _ in range(2)]
    with pytest.raises(_lib.BMError, match="head_dim"):
        ops.PagedKV8(**tensors(k_pages=pages[0], v_pages=pages[1]))


def test_python_calls_refuse_cpu_tensors_and_missing_arguments():
    x, w = torch.zeros(2, 4, 64), torch.ones(64)
    table = type("Table", (), dict(data=torch.zeros(4, 32, 2), max_pos=4, head_dim=64))
    for args in ((x, None, w, None, 0, table), (x, None, w, None, None, table), (x, None, w, None, 0, None),
                 (None, None, None, None, 0, table)):
        with pytest.raises(_lib.BMError):
            ops.qk_norm_rotary(*args)
    c = type("Cache", (), {**tensors(), "num_kv_heads": 2, "head_dim": 64, "device": torch.device("cpu")})
    lens = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.BMError):
        ops.paged_kv8_append(None, x[:, :2], x[:, 2:], c, lens, torch.zeros(3, dtype=torch.int32), 1)
    with pytest.raises(_lib.BMError):
        ops.paged_kv8_read(c, lens, torch.zeros(3, dtype=torch.int32), 2, 1)
    with pytest.raises(_lib.BMError):
        ops.paged_kv8_read(c, lens, torch.zeros(3, dtype=torch.int32), -1, 1)
    with pytest.raises(_lib.BMError):
        ops.paged_kv8_read(c, lens, torch.zeros(3, dtype=torch.int32), 2, 1, k_out=torch.zeros(2, 2, 32))


def test_the_plain_form_encodes_as_the_format_says():
    """kv8_ref's codes against torch's conversion, and its exponents against logarithms."""
    x = torch.randn(20000, generator=torch.Generator().manual_seed(1)) * torch.exp2(torch.arange(20000) % 24 - 14.0)
    x = x.clamp(-448, 448)
    assert np.array_equal(kv8_ref.encode(x.double().numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    codes = np.arange(256, dtype=np.uint8)
    assert np.array_equal(kv8_ref.VALUES, torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    for a in [448.0, 448.0000001, 447.9, 1.75, 1.7500001, 1.0, 3e-5, 0.0, 1e30, 1e-30]:
        want = -40 if a == 0 else min(max(int(np.ceil(np.log2(a / 448.0))), -40), 40)
        assert kv8_ref.exponent(a) == want
