"""CPU-side refusals of the paged-cache serving entry points: bad arguments are rejected on
the host before anything reaches CUDA, empty calls do nothing, and the ctypes structs
mirror the header's."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from baremetalinferenceengine_b200 import _lib, build, ops

FAKE = 0x1000000  # never dereferenced: every call below fails or returns before any CUDA call
FAR = 0x4000000


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def cache(**kw):
    c = dict(k_pages=FAKE, v_pages=FAKE, page_table=FAKE, num_pages=4, page_size=8, max_pages=2, num_seqs=2,
             num_kv_heads=2, head_dim=64)
    c.update(kw)
    return ctypes.byref(_lib.PagedKVC(*[c[n] for n, _ in _lib.PagedKVC._fields_]))


def fill(L, table=FAKE, max_pos=8, dim=64, theta=1e4, **s):
    full = dict(kind=0, original_max_pos=512, factor=2.0, low=1.0, high=4.0, mscale=0.0)
    full.update(s)
    return L.bm_rotary_table_fill(table, max_pos, dim, theta, ctypes.byref(_lib.RopeScalingC(**full)), None)


def rotary(L, qo=FAR, ko=FAR * 2, q=FAKE, k=FAKE * 2, pos=FAKE, pos0=0, table=FAKE, n=8, rd=64, rows=4, hq=4, hkv=2,
           hd=64, qs=256, ks=128, qos=256, kos=128, dtype=0):
    return L.bm_rotary(qo, ko, q, k, pos, pos0, table, n, rd, 0, rows, hq, hkv, hd, qs, ks, qos, kos, dtype, None, None)


def append(L, qo=FAR, q=FAKE, k=FAKE * 2, v=FAKE * 3, pos=FAKE, slots=None, c=None, table=FAKE, n=8, rd=64, rows=4, hq=4,
           qs=256, ks=128, vs=128, qos=256, dtype=0):
    return L.bm_paged_kv_append(qo, q, k, v, pos, slots, None, c or cache(), table, n, rd, 0, rows, hq, qs, ks, vs, qos,
                                dtype, None, None)


def attend(L, out=FAR, q=FAKE, c=None, ctx=FAKE, starts=FAKE, mask=FAKE, words=1, total=4, batch=2, hq=4, max_ctx=8,
           max_tree=4, scale=0.0, ws=FAR * 4, ws_bytes=1 << 40, dtype=0, seqs=None):
    return L.bm_paged_tree_attention(out, q, c or cache(), seqs, ctx, starts, mask, words, total, batch, hq, max_ctx,
                                     max_tree, scale, ws, ws_bytes, dtype, None, None)


def size(L, total=4, batch=2, hq=4, hkv=2, hd=64, max_ctx=8, max_tree=4, out=True):
    return L.bm_paged_tree_attention_workspace_size(total, batch, hq, hkv, hd, max_ctx, max_tree,
                                                    ctypes.byref(ctypes.c_size_t()) if out else None)


def sample(L, tokens=FAKE, logits=FAKE, u=FAKE, rows=2, vocab=10, stride=10, dtype=0):
    return L.bm_sample(tokens, logits, u, None, None, None, None, rows, vocab, stride, dtype, None, None)


@pytest.mark.parametrize("call", [
    lambda L: fill(L, max_pos=0), lambda L: fill(L, dim=7), lambda L: fill(L, dim=0), lambda L: fill(L, theta=0.0),
    lambda L: fill(L, theta=float("inf")), lambda L: fill(L, table=None), lambda L: fill(L, table=FAKE + 4),
    lambda L: fill(L, kind=5), lambda L: fill(L, kind=-1), lambda L: fill(L, kind=1, factor=0.5),
    lambda L: fill(L, kind=1, factor=float("nan")), lambda L: fill(L, kind=2, dim=2),
    lambda L: fill(L, kind=3, low=4.0, high=4.0), lambda L: fill(L, kind=3, original_max_pos=0),
    lambda L: fill(L, kind=4, low=1.0, high=2.0), lambda L: fill(L, kind=4, low=32.0, high=0.0),
    lambda L: fill(L, kind=4, low=32.0, high=1.0, theta=1.0), lambda L: fill(L, mscale=float("nan")),
    lambda L: rotary(L, dtype=3), lambda L: rotary(L, rows=-1), lambda L: rotary(L, hq=-1),
    lambda L: rotary(L, table=None), lambda L: rotary(L, n=0), lambda L: rotary(L, table=FAKE + 4),
    lambda L: rotary(L, rd=7), lambda L: rotary(L, rd=0), lambda L: rotary(L, rd=66), lambda L: rotary(L, hd=1026),
    lambda L: rotary(L, q=None), lambda L: rotary(L, ko=None), lambda L: rotary(L, qs=255), lambda L: rotary(L, kos=64),
    lambda L: rotary(L, pos=None, pos0=-1), lambda L: rotary(L, pos=None, pos0=2 ** 31 - 3),
    lambda L: rotary(L, qo=FAKE + 4),                       # overlaps q without being it
    lambda L: rotary(L, qo=FAKE, qos=300),                  # q's pointer, another stride
    lambda L: rotary(L, qo=FAKE * 2),                       # q_out over k
    lambda L: rotary(L, ko=FAR + 16),                       # both outputs in one place
    lambda L: rotary(L, q=FAKE, k=FAKE + 255 * 4, qs=400, ks=400, qo=FAKE, qos=400),  # k begins in q's last head
    lambda L: append(L, dtype=2), lambda L: append(L, rows=-2), lambda L: append(L, k=None), lambda L: append(L, v=None),
    lambda L: append(L, q=None), lambda L: append(L, qo=None), lambda L: append(L, pos=None),
    lambda L: append(L, pos=None, slots=FAKE),              # rotation wants positions
    lambda L: append(L, pos=None, table=None), lambda L: append(L, n=0), lambda L: append(L, rd=65),
    lambda L: append(L, rd=128), lambda L: append(L, ks=127), lambda L: append(L, vs=0), lambda L: append(L, qos=1),
    lambda L: append(L, qo=FAKE + 16), lambda L: append(L, qo=FAKE * 3),
    lambda L: append(L, c=cache(k_pages=None)), lambda L: append(L, c=cache(page_table=None)),
    lambda L: append(L, c=cache(num_pages=0)), lambda L: append(L, c=cache(page_size=0)),
    lambda L: append(L, c=cache(max_pages=-1)), lambda L: append(L, c=cache(num_seqs=0)),
    lambda L: append(L, c=cache(num_kv_heads=0)), lambda L: append(L, c=cache(head_dim=2048)),
    lambda L: append(L, c=cache(page_size=1 << 20, max_pages=1 << 12)),  # slots past int32
    lambda L: L.bm_paged_kv_append(FAR, FAKE, FAKE, FAKE, FAKE, None, None, None, None, 0, 0, 0, 1, 1, 64, 64, 64, 64, 0,
                                   None, None),
    lambda L: attend(L, dtype=9), lambda L: attend(L, c=cache(page_size=0)), lambda L: attend(L, total=-1),
    lambda L: attend(L, batch=-1), lambda L: attend(L, hq=3), lambda L: attend(L, hq=0), lambda L: attend(L, hq=130),
    lambda L: attend(L, c=cache(head_dim=260)), lambda L: attend(L, c=cache(head_dim=66)),
    lambda L: attend(L, c=cache(head_dim=60), dtype=1), lambda L: attend(L, max_ctx=-1), lambda L: attend(L, max_tree=-1),
    lambda L: attend(L, max_ctx=1 << 30), lambda L: attend(L, words=0), lambda L: attend(L, max_tree=65),
    lambda L: attend(L, scale=float("nan")), lambda L: attend(L, out=None), lambda L: attend(L, q=None),
    lambda L: attend(L, ctx=None), lambda L: attend(L, starts=None), lambda L: attend(L, q=FAKE + 4),
    lambda L: attend(L, out=FAR + 8), lambda L: attend(L, ws=FAR + 4), lambda L: attend(L, out=FAKE + 64),
    lambda L: attend(L, batch=3),                            # more sequences than the cache's two
    lambda L: attend(L, ws=None, max_ctx=4096), lambda L: attend(L, ws_bytes=64, max_ctx=4096),
    lambda L: size(L, out=False), lambda L: size(L, hd=0), lambda L: size(L, hq=5), lambda L: size(L, total=-1),
    lambda L: size(L, batch=1 << 20, max_tree=1 << 10),
    lambda L: sample(L, dtype=4), lambda L: sample(L, rows=-1), lambda L: sample(L, vocab=0), lambda L: sample(L, stride=9),
    lambda L: sample(L, vocab=(1 << 24) + 1, stride=1 << 25), lambda L: sample(L, tokens=None),
    lambda L: sample(L, logits=None), lambda L: sample(L, u=None),
])
def test_host_checks_reject_before_any_launch(lib, call):
    assert call(lib) == _lib.BM_ERR_INVALID_ARGUMENT
    assert lib.bm_last_error_message()


@pytest.mark.parametrize("call", [
    lambda L: rotary(L, rows=0), lambda L: rotary(L, hq=0, hkv=0), lambda L: append(L, rows=0),
    lambda L: attend(L, batch=0), lambda L: attend(L, total=0), lambda L: attend(L, max_tree=0), lambda L: size(L, batch=0),
    lambda L: sample(L, rows=0),
])
def test_empty_calls_are_no_ops(lib, call):
    assert call(lib) == _lib.BM_OK


@pytest.mark.parametrize("struct,name", [(_lib.PagedKVC, "bm_paged_kv_t"), (_lib.RopeScalingC, "bm_rope_scaling_t")])
def test_struct_layouts_match_the_header(struct, name):
    fields = [f for f, _ in struct._fields_]
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "bm_layer_ops.h"\nint main(void) {\n'
    src += f'  printf("%zu\\n", sizeof({name}));\n'
    src += "".join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "  return 0;\n}\n"
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = os.path.join(tmp, "layout.c"), os.path.join(tmp, "layout")
        with open(c, "w") as fh:
            fh.write(src)
        inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
        subprocess.run(["gcc", "-std=c11", "-I", inc, "-o", exe, c], check=True)
        out = [int(x) for x in subprocess.run([exe], capture_output=True, text=True).stdout.split()]
    assert out == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def test_python_layer_rejects_cpu_tensors_and_bad_arguments():
    x = torch.zeros(2, 4, 64)
    pos = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.BMError):
        ops.rotary(None, None, pos, None)
    with pytest.raises(_lib.BMError):
        ops.rotary(x, None, pos, None)  # no CPU path
    with pytest.raises(_lib.BMError):
        ops.PagedKV(torch.zeros(2, 2, 8, 64), torch.zeros(2, 2, 8, 64), pos[None])
    with pytest.raises(_lib.BMError):
        ops.PagedKV(torch.zeros(2, 2, 8, 64), torch.zeros(2, 2, 4, 64), pos[None])
    with pytest.raises(_lib.BMError):
        ops.sample(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(_lib.BMError):
        ops.RopeScaling("stretch", 2.0).c_struct()
    with pytest.raises(_lib.BMError):
        ops.RopeScaling("linear", 2.0, mscale=-1.0).c_struct()


MISALIGNED = {
    "rotary": [dict(q=FAKE + 2), dict(k=FAKE * 2 + 1), dict(qo=FAR + 3), dict(ko=FAR * 2 + 2), dict(pos=FAKE + 2),
               dict(q=FAKE + 1, dtype=1), dict(ko=FAR * 2 + 1, dtype=1)],
    "append": [dict(q=FAKE + 2), dict(k=FAKE * 2 + 2), dict(v=FAKE * 3 + 1), dict(qo=FAR + 2), dict(pos=FAKE + 1),
               dict(slots=FAKE + 2), dict(v=FAKE * 3 + 1, dtype=1), dict(k_pages=FAKE + 2), dict(v_pages=FAKE + 1),
               dict(v_pages=FAKE + 1, dtype=1), dict(page_table=FAKE + 2)],
    "attend": [dict(ctx=FAKE + 2), dict(starts=FAKE + 1), dict(mask=FAKE + 4), dict(seqs=FAKE + 2), dict(page_table=FAKE + 2)],
    "sample": [dict(logits=FAKE + 2), dict(logits=FAKE + 1, dtype=1), dict(tokens=FAKE + 2), dict(u=FAKE + 1)],
}


@pytest.mark.parametrize("name,kw", [(n, kw) for n, all_kw in MISALIGNED.items() for kw in all_kw])
def test_pointers_below_their_elements_alignment_are_refused(lib, name, kw):
    """A kernel's scalar loads need it, too: such a pointer would fault there."""
    kw = dict(kw)
    in_cache = {f: kw.pop(f) for f in ("k_pages", "v_pages", "page_table") if f in kw}
    call = {"rotary": rotary, "append": append, "attend": attend, "sample": sample}[name]
    assert call(lib, **kw, **({"c": cache(**in_cache)} if in_cache else {})) == _lib.BM_ERR_INVALID_ARGUMENT
    assert b"aligned" in lib.bm_last_error_message()


# pages of 4 * 2 * 8 * 64 elements: 16 KB in fp32, 8 KB in bf16
@pytest.mark.parametrize("name,kw", [
    ("append", dict(k_pages=FAR)), ("append", dict(v_pages=FAR)), ("append", dict(v_pages=FAR - 16380)),
    ("append", dict(k_pages=FAR + 4 * 4 * 64 * 4 - 4)), ("append", dict(k_pages=FAR - 8190, dtype=1)),
    ("attend", dict(k_pages=FAR)), ("attend", dict(v_pages=FAR + 4080)), ("attend", dict(v_pages=FAR - 16368))])
def test_outputs_over_the_cache_are_refused(lib, name, kw):
    kw = dict(kw)
    dtype = kw.pop("dtype", 0)
    call = {"append": append, "attend": attend}[name]
    assert call(lib, c=cache(**kw), dtype=dtype) == _lib.BM_ERR_INVALID_ARGUMENT
    assert b"pages" in lib.bm_last_error_message()


def test_rotary_without_positions_is_refused():
    """None is no pos0 of 0."""
    table = type("Table", (), dict(data=torch.zeros(4, 32, 2), max_pos=4, head_dim=64))
    with pytest.raises(_lib.BMError, match="positions"):
        ops.rotary(torch.zeros(2, 4, 64), None, None, table)


@pytest.mark.parametrize("scale", [float("inf"), 3.4e38, float("nan")])
def test_a_scale_that_is_not_finite_is_refused(lib, scale):
    """Times log2(e), too: every output would be NaN."""
    assert attend(lib, scale=scale) == _lib.BM_ERR_INVALID_ARGUMENT
    assert b"scale" in lib.bm_last_error_message()
