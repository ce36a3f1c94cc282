"""Host-side API over the C ABI, on torch CUDA tensors (torch provides device
memory and streams; every op runs in ``libbm_layer_ops.so``).

Two layers, mirroring the reference:

* ``launch_*`` — the reference's single-token fp32 launch functions
  (include/kernels.cuh:9,15,29,32,36) with the same names, argument order and
  meaning; tensors stand in for the raw device pointers. Where the reference
  exits the process through CUDA_CHECK, these raise :class:`BMError`.
* batched ops — ``embed_gather``, ``rmsnorm``, ``add_rmsnorm``, ``swiglu``,
  ``add``, ``rope``, ``rope_kv_store``, ``kv_store`` over many rows, fp32 or
  bf16, on the current torch stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
import dataclasses
from typing import Optional

import torch

from . import _lib
from ._lib import BMError, check, load  # noqa: F401  (re-exported)

_DTYPES = {torch.float32: _lib.BM_F32, torch.bfloat16: _lib.BM_BF16}


def bm_dtype(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, f"unsupported dtype {t.dtype} (float32 or bfloat16)") from None


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    if t is None:
        return None
    if not t.is_cuda:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "tensor is not on a CUDA device")
    return t.data_ptr()


def _dev(t: torch.Tensor) -> torch.device:
    """The tensor's CUDA device; a CPU tensor is an argument error (no CPU path)."""
    if not t.is_cuda:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "tensor is not on a CUDA device")
    return t.device


def _stream(device: torch.device, stream: Optional[torch.cuda.Stream]) -> int:
    s = stream if stream is not None else torch.cuda.current_stream(device)
    return s.cuda_stream


def _dense(t: torch.Tensor, name: str) -> None:
    if not t.is_contiguous():
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, f"{name} must be contiguous")


def _same(ref: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    for o in others:
        if o is not None and (o.device != ref.device or o.dtype != ref.dtype):
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "tensors must share device and dtype")


def _i32(t: Optional[torch.Tensor], name: str) -> None:
    if t is not None and (t.dtype != torch.int32 or not t.is_contiguous() or not t.is_cuda):
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, f"{name} must be a contiguous int32 CUDA tensor")


class DeviceStatus:
    """One int32 device word that kernels OR ``BM_DEVERR_*`` bits into."""

    def __init__(self, device: torch.device | str | int = "cuda"):
        self.word = torch.zeros(1, dtype=torch.int32, device=device)

    @property
    def ptr(self) -> int:
        return self.word.data_ptr()

    def read(self, stream: Optional[torch.cuda.Stream] = None) -> int:
        """Synchronises the stream, returns the bits and clears the word."""
        flags = ctypes.c_int32(0)
        with torch.cuda.device(self.word.device):
            st = load().bm_status_read(self.ptr, ctypes.byref(flags), _stream(self.word.device, stream))
        if st not in (_lib.BM_OK, _lib.BM_ERR_DEVICE):
            check(st)
        return int(flags.value)


@dataclasses.dataclass(frozen=True)
class RopeScaling:
    """How a :class:`RopeTable` stretches its frequencies for contexts past the trained
    one (the formulas stand at bm_rotary_table_fill): ``kind`` none, linear, ntk, bands
    (low_freq_factor, high_freq_factor) or yarn (beta_fast, beta_slow). ``mscale``
    multiplies cos and sin; None is the kind's own (0.1 ln(factor) + 1 for yarn)."""

    kind: str = "none"
    factor: float = 1.0
    original_max_pos: int = 0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    mscale: Optional[float] = None

    def c_struct(self) -> "_lib.RopeScalingC":
        if self.kind not in _lib.BM_ROPE_SCALING:
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, f"unknown rope scaling {self.kind!r}")
        if self.mscale is not None and not self.mscale > 0:
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "mscale must be > 0")
        yarn = self.kind == "yarn"
        return _lib.RopeScalingC(_lib.BM_ROPE_SCALING[self.kind], int(self.original_max_pos), float(self.factor),
                                 float(self.beta_fast if yarn else self.low_freq_factor),
                                 float(self.beta_slow if yarn else self.high_freq_factor),
                                 0.0 if self.mscale is None else float(self.mscale))


class RopeTable:
    """Device (cos, sin) table [max_pos][head_dim/2] of fp32 pairs, filled in fp64; with
    ``scaling`` (a :class:`RopeScaling`) its frequencies stretched. For heads that are
    rotated in part, ``head_dim`` is the rotated part (rotary, paged_kv_append)."""

    def __init__(self, max_pos: int, head_dim: int, theta: float, device: torch.device | str | int = "cuda",
                 stream: Optional[torch.cuda.Stream] = None, scaling: Optional[RopeScaling] = None):
        self.max_pos, self.head_dim, self.theta = int(max_pos), int(head_dim), float(theta)
        self.scaling = scaling
        self.data = torch.empty(self.max_pos, self.head_dim // 2, 2, dtype=torch.float32, device=device)
        with torch.cuda.device(self.data.device):
            s = _stream(self.data.device, stream)
            if scaling is None:
                check(load().bm_rope_table_fill(self.data.data_ptr(), self.max_pos, self.head_dim, self.theta, s))
            else:
                check(load().bm_rotary_table_fill(self.data.data_ptr(), self.max_pos, self.head_dim, self.theta,
                                                  ctypes.byref(scaling.c_struct()), s))

    @property
    def ptr(self) -> int:
        return self.data.data_ptr()


# --------------------------------------------------------------------------
# Batched ops
# --------------------------------------------------------------------------

def embed_gather(table: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None,
                 status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """out[r] = table[ids[r]] (bit-exact). Bad ids leave rows unwritten and set BAD_ID."""
    _dense(table, "table")
    _i32(ids, "ids")
    rows, (vocab, dim) = ids.numel(), table.shape
    if out is None:
        out = torch.empty(rows, dim, dtype=table.dtype, device=table.device)
    _same(table, out)
    if out.dim() != 2 or out.shape[0] != rows or out.shape[1] != dim or out.stride(1) != 1:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "out must be [rows, dim] with unit inner stride")
    with torch.cuda.device(_dev(table)):
        check(load().bm_embed_gather(_ptr(out), _ptr(table), _ptr(ids), rows, dim, vocab, out.stride(0),
                                     bm_dtype(table), status.ptr if status else None,
                                     _stream(table.device, stream)))
    return out


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5, out: Optional[torch.Tensor] = None,
            stream=None) -> torch.Tensor:
    """Row-wise RMSNorm of x [rows, dim]; ``out=x`` normalises in place."""
    dim = x.shape[-1]
    x2 = x.reshape(-1, dim) if x.is_contiguous() else x
    if x2.dim() != 2 or x2.stride(1) != 1:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "x must be [rows, dim] with unit inner stride")
    if out is None:
        out = torch.empty_like(x)
    out2 = out.reshape(-1, dim) if out.is_contiguous() else out
    _same(x, weight, out)
    if weight.numel() != dim:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "weight must have dim elements")
    with torch.cuda.device(_dev(x)):
        check(load().bm_rmsnorm(_ptr(out2), _ptr(x2), _ptr(weight), x2.shape[0], dim, eps, x2.stride(0),
                                out2.stride(0), bm_dtype(x), _stream(x.device, stream)))
    return out


def add_rmsnorm(residual: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """residual += delta (in place); returns rmsnorm(residual) * weight."""
    for t, n in ((residual, "residual"), (delta, "delta")):
        _dense(t, n)
    if residual.shape != delta.shape:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "residual and delta shapes differ")
    dim = residual.shape[-1]
    if out is None:
        out = torch.empty_like(residual)
    _dense(out, "out")
    _same(residual, delta, weight, out)
    with torch.cuda.device(_dev(residual)):
        check(load().bm_add_rmsnorm(_ptr(residual), _ptr(delta), _ptr(weight), _ptr(out), residual.numel() // dim,
                                    dim, eps, bm_dtype(residual), _stream(residual.device, stream)))
    return out


def swiglu(gate: torch.Tensor, up: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out = silu(gate) * up, element-wise."""
    _dense(gate, "gate")
    _dense(up, "up")
    if out is None:
        out = torch.empty_like(gate)
    _dense(out, "out")
    _same(gate, up, out)
    if gate.numel() != up.numel() or out.numel() != gate.numel():
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "gate, up and out sizes differ")
    with torch.cuda.device(_dev(gate)):
        check(load().bm_swiglu(_ptr(out), _ptr(gate), _ptr(up), gate.numel(), bm_dtype(gate),
                               _stream(gate.device, stream)))
    return out


def add(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """out = a + b, element-wise (out may be a or b)."""
    _dense(a, "a")
    _dense(b, "b")
    if out is None:
        out = torch.empty_like(a)
    _dense(out, "out")
    _same(a, b, out)
    if a.numel() != b.numel() or out.numel() != a.numel():
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "a, b and out sizes differ")
    with torch.cuda.device(_dev(a)):
        check(load().bm_add(_ptr(out), _ptr(a), _ptr(b), a.numel(), bm_dtype(a), _stream(a.device, stream)))
    return out


def gemm_swiglu(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, out: Optional[torch.Tensor] = None,
                status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """out = silu(x @ w_gate) * (x @ w_up): x [rows, dim], w_gate and w_up [dim, hidden]
    (the reference's [in][out] weight layout). bf16 on the tensor cores; fp32 on CUDA
    cores (the SwiGLU of bm_swiglu applied to the reduced products)."""
    for t, name in ((x, "x"), (w_gate, "w_gate"), (w_up, "w_up")):
        _dense(t, name)
    if x.dim() != 2 or w_gate.dim() != 2 or w_gate.shape != w_up.shape or w_gate.shape[0] != x.shape[1]:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need x [rows, dim] and w_gate, w_up [dim, hidden]")
    rows, dim = x.shape
    hidden = w_gate.shape[1]
    if out is None:
        out = torch.empty((rows, hidden), dtype=x.dtype, device=x.device)
    _dense(out, "out")
    _same(x, w_gate, w_up, out)
    if tuple(out.shape) != (rows, hidden):
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "out must be [rows, hidden]")
    with torch.cuda.device(_dev(x)):
        check(load().bm_gemm_swiglu(_ptr(out), _ptr(x), _ptr(w_gate), _ptr(w_up), rows, dim, hidden, bm_dtype(x),
                                    status.ptr if status else None, _stream(x.device, stream)))
    return out


def gemm(a: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None,
         status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """out = a @ b: a [m, k], b [k, n] (launch_gemm's operand layout). bf16 runs on
    the tensor cores; fp32 on CUDA cores (built for few rows)."""
    _dense(a, "a")
    _dense(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need a [m, k] and b [k, n]")
    m, k = a.shape
    n = b.shape[1]
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _dense(out, "out")
    _same(a, b, out)
    if tuple(out.shape) != (m, n):
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "out must be [m, n]")
    with torch.cuda.device(_dev(a)):
        check(load().bm_gemm(_ptr(out), _ptr(a), _ptr(b), m, n, k, bm_dtype(a), status.ptr if status else None,
                             _stream(a.device, stream)))
    return out


def gemm_shared_a(a: torch.Tensor, bs, outs=None, status: Optional[DeviceStatus] = None, stream=None):
    """[a @ b for b in bs] for one to three weights b [k, n_o] (an attention block's Q,
    K and V projections): fp32 in one launch, bf16 one tensor-core GEMM per weight."""
    _dense(a, "a")
    bs = list(bs)
    if not 1 <= len(bs) <= 3:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "one to three weights")
    if a.dim() != 2:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need a [m, k]")
    m, k = a.shape
    for b in bs:
        _dense(b, "b")
        if b.dim() != 2 or b.shape[0] != k:
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need every b [k, n]")
    if outs is None:
        outs = [torch.empty((m, b.shape[1]), dtype=a.dtype, device=a.device) for b in bs]
    outs = list(outs)
    for b, out in zip(bs, outs):
        _dense(out, "out")
        if tuple(out.shape) != (m, b.shape[1]):
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "every out must be [m, n]")
    _same(a, *bs, *outs)
    count = len(bs)
    c_arr = (ctypes.c_void_p * count)(*[_ptr(o) for o in outs])
    b_arr = (ctypes.c_void_p * count)(*[_ptr(b) for b in bs])
    n_arr = (ctypes.c_int32 * count)(*[b.shape[1] for b in bs])
    with torch.cuda.device(_dev(a)):
        check(load().bm_gemm_shared_a(c_arr, _ptr(a), b_arr, n_arr, count, m, k, bm_dtype(a),
                                      status.ptr if status else None, _stream(a.device, stream)))
    return outs


def rmsnorm_gemm(h: torch.Tensor, norm_weight: torch.Tensor, bs, d: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 swiglu: bool = False, outs=None, residual_out: Optional[torch.Tensor] = None,
                 normed: Optional[torch.Tensor] = None, status: Optional[DeviceStatus] = None, stream=None):
    """The norm before a projection and the projection: y = rmsnorm(h + d) * norm_weight
    (d optional), then [y @ b for b in bs] (one to three weights), or with swiglu
    (bs = [w_gate, w_up]) the one output silu(y @ w_gate) * (y @ w_up). residual_out,
    when given with d, receives h + d. fp32 rows that fit run as one launch."""
    _dense(h, "h")
    bs = list(bs)
    if h.dim() != 2:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need h [m, k]")
    m, k = h.shape
    if (len(bs) != 2) if swiglu else not 1 <= len(bs) <= 3:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "two weights with swiglu, else one to three")
    for b in bs:
        _dense(b, "b")
        if b.dim() != 2 or b.shape[0] != k:
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "need every b [k, n]")
    widths = [b.shape[1] for b in bs]
    n_out = 1 if swiglu else len(bs)
    if outs is None:
        outs = [torch.empty((m, widths[o]), dtype=h.dtype, device=h.device) for o in range(n_out)]
    outs = list(outs)
    if len(outs) != n_out:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "one output per product (one with swiglu)")
    for o, out in enumerate(outs):
        _dense(out, "out")
        if tuple(out.shape) != (m, widths[o]):
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "every out must be [m, n]")
    if normed is None:
        normed = torch.empty_like(h)
    extra = [t for t in (d, residual_out) if t is not None]
    for t in extra + [normed]:
        _dense(t, "h-shaped tensor")
        if tuple(t.shape) != (m, k):
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "d, residual_out and normed must be [m, k]")
    _dense(norm_weight, "norm_weight")
    _same(h, norm_weight, *bs, *outs, normed, *extra)
    count = len(bs)
    c_arr = (ctypes.c_void_p * count)(*([_ptr(o) for o in outs] + [None] * (count - len(outs))))
    b_arr = (ctypes.c_void_p * count)(*[_ptr(b) for b in bs])
    n_arr = (ctypes.c_int32 * count)(*widths)
    with torch.cuda.device(_dev(h)):
        check(load().bm_rmsnorm_gemm(c_arr, _ptr(h), _ptr(d), _ptr(norm_weight), eps,
                                     _ptr(residual_out), _ptr(normed), b_arr,
                                     n_arr, count, int(swiglu), m, k, bm_dtype(h), status.ptr if status else None,
                                     _stream(h.device, stream)))
    return outs


def softmax(x: torch.Tensor, size: Optional[int] = None, num_vectors: int = 1, stride: Optional[int] = None,
            stream=None) -> torch.Tensor:
    """In place: num_vectors vectors of `size` elements, `stride` apart, each
    replaced by exp(x - max) / sum exp(x - max) (defaults: x as one vector)."""
    _dense(x, "x")
    size = x.numel() if size is None else size
    stride = size if stride is None else stride
    if num_vectors > 0 and size > 0 and (num_vectors - 1) * stride + size > x.numel():
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "vectors reach past x")
    with torch.cuda.device(_dev(x)):
        check(load().bm_softmax(_ptr(x), size, num_vectors, stride, bm_dtype(x), _stream(x.device, stream)))
    return x


def _positions(positions, rows):
    if isinstance(positions, int):
        return None, positions
    _i32(positions, "positions")
    if positions.numel() != rows:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "positions must have one entry per row")
    return positions, 0


def rope_kv_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, table: Optional[RopeTable] = None, theta: float = 10000.0,
                  seq_ids: Optional[torch.Tensor] = None, status: Optional[DeviceStatus] = None,
                  stream=None) -> None:
    """Rotates q [rows, Hq, hd] in place; writes rotated k and raw v into the caches
    [num_seqs, Hkv, max_seq, hd] at (seq_ids[r], positions[r]). ``positions`` is an
    int32 tensor or an int pos0 (token r at pos0 + r)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _dense(t, n)
    _same(q, k, v, k_cache, v_cache)
    rows, hq, hd = q.shape[0], q.shape[1], q.shape[2]
    hkv = k.shape[1]
    num_seqs, max_seq = k_cache.shape[0], k_cache.shape[2]
    if k.shape != v.shape or k.shape[0] != rows or k_cache.shape != v_cache.shape or k_cache.shape[1] != hkv:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "q/k/v/cache shapes disagree")
    pos_t, pos0 = _positions(positions, rows)
    _i32(seq_ids, "seq_ids")
    with torch.cuda.device(_dev(q)):
        check(load().bm_rope_kv_store(_ptr(q), _ptr(k), _ptr(v), _ptr(pos_t), pos0, _ptr(seq_ids), _ptr(k_cache),
                                      _ptr(v_cache), table.ptr if table else None,
                                      table.max_pos if table else 0, theta, rows, hq, hkv, hd, max_seq, num_seqs,
                                      bm_dtype(q), status.ptr if status else None, _stream(q.device, stream)))


def rope(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions, table: Optional[RopeTable] = None,
         theta: float = 10000.0, status: Optional[DeviceStatus] = None, stream=None) -> None:
    """Rotates q [rows, Hq, hd] and k [rows, Hkv, hd] in place (either may be None)."""
    ref = q if q is not None else k
    for t, n in ((q, "q"), (k, "k")):
        if t is not None:
            _dense(t, n)
    _same(ref, q, k)
    rows, hd = ref.shape[0], ref.shape[2]
    pos_t, pos0 = _positions(positions, rows)
    with torch.cuda.device(_dev(ref)):
        check(load().bm_rope(_ptr(q), _ptr(k), _ptr(pos_t), pos0, table.ptr if table else None,
                             table.max_pos if table else 0, theta, rows, q.shape[1] if q is not None else 0,
                             k.shape[1] if k is not None else 0, hd, bm_dtype(ref),
                             status.ptr if status else None, _stream(ref.device, stream)))


def kv_store(cache: torch.Tensor, src: torch.Tensor, positions, seq_ids: Optional[torch.Tensor] = None,
             status: Optional[DeviceStatus] = None, stream=None) -> None:
    """cache [num_seqs, H, max_seq, hd][seq_ids[r], :, positions[r]] = src [rows, H, hd][r]."""
    _dense(cache, "cache")
    _dense(src, "src")
    _same(cache, src)
    rows, h, hd = src.shape
    pos_t, pos0 = _positions(positions, rows)
    _i32(seq_ids, "seq_ids")
    with torch.cuda.device(_dev(src)):
        check(load().bm_kv_store(_ptr(cache), _ptr(src), _ptr(pos_t), pos0, _ptr(seq_ids), rows, h, hd,
                                 cache.shape[2], cache.shape[0], bm_dtype(src), status.ptr if status else None,
                                 _stream(src.device, stream)))


# --------------------------------------------------------------------------
# Rotary forms, the paged KV cache, tree attention and sampling
# --------------------------------------------------------------------------

def _invalid(message: str) -> BMError:
    return BMError(_lib.BM_ERR_INVALID_ARGUMENT, message)


def _empty(shape, dtype: torch.dtype, device: torch.device, stream) -> torch.Tensor:
    """Uninitialised memory that belongs to the stream that will write it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _like(t: Optional[torch.Tensor], stream):
    """Room for an output like `t`, made on the stream that will write it."""
    return _empty(t.shape, t.dtype, t.device, stream)


def _word(status: Optional[DeviceStatus]) -> Optional[torch.Tensor]:
    return None if status is None else status.word


def _handle(stream: Optional[torch.cuda.Stream]) -> Optional[int]:
    """A stream's handle; None is the current stream of the tensors' device."""
    return None if stream is None else stream.cuda_stream


def rotary(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions, table: RopeTable,
           interleaved: bool = False, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
           status: Optional[DeviceStatus] = None, stream=None):
    """Rotates the first ``table.head_dim`` elements of every head of q [rows, Hq, hd] and
    k [rows, Hkv, hd] (either may be None) and copies the rest; returns (q_out, k_out),
    made when not given; ``q_out=q`` rotates in place. Pairs are (i, i + rotary_dim/2),
    or (2i, 2i + 1) with ``interleaved``. q and k may be slices of a fused projection's
    rows. ``positions``: int32 tensor, or an int pos0 (row r at pos0 + r). A position
    outside the table leaves its row unwritten and sets BAD_POSITION."""
    if table is None:
        raise _invalid("rotary needs a table")
    if positions is None:
        raise _invalid("rotary needs positions")
    if stream is not None:
        q_out = _like(q, stream) if q is not None and q_out is None else q_out
        k_out = _like(k, stream) if k is not None and k_out is None else k_out
    pos, pos0 = (None, positions) if isinstance(positions, int) else (positions, 0)
    return _lib.serving_ops().rotary(q, k, pos, pos0, table.data, table.max_pos, table.head_dim, interleaved, q_out, k_out,
                                     _word(status), _handle(stream))


class PagedKV:
    """A paged KV cache over the caller's tensors: k_pages and v_pages [num_pages, Hkv,
    page_size, hd] (contiguous, one dtype and device) and page_table int32 [num_seqs,
    max_pages]: slot t of sequence s is in page page_table[s, t // page_size] at
    t % page_size. Every call reads (and checks) the three tensors that the object holds then:
    page_table may be rewritten between calls (on the calls' stream), and each may be replaced
    by another."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise _invalid("k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim]")
        _dense(k_pages, "k_pages")
        _dense(v_pages, "v_pages")
        bm_dtype(k_pages)
        _same(k_pages, v_pages)
        if page_table.dim() != 2:
            raise _invalid("page_table must be [num_seqs, max_pages]")
        if page_table.dtype != torch.int32 or not page_table.is_contiguous() or page_table.device != _dev(k_pages):
            raise _invalid("page_table must be a contiguous int32 tensor on the pages' device")
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table

    num_pages = property(lambda self: self.k_pages.shape[0])
    num_kv_heads = property(lambda self: self.k_pages.shape[1])
    page_size = property(lambda self: self.k_pages.shape[2])
    head_dim = property(lambda self: self.k_pages.shape[3])
    num_seqs = property(lambda self: self.page_table.shape[0])
    max_pages = property(lambda self: self.page_table.shape[1])
    device = property(lambda self: self.k_pages.device)
    dtype = property(lambda self: self.k_pages.dtype)


def paged_kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, positions: Optional[torch.Tensor],
                    cache: PagedKV, table: Optional[RopeTable] = None, seq_ids: Optional[torch.Tensor] = None,
                    slots: Optional[torch.Tensor] = None, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None, status: Optional[DeviceStatus] = None,
                    stream=None) -> Optional[torch.Tensor]:
    """rope_kv_store for a paged cache: writes rotated k and raw v [rows, Hkv, hd] into
    slot ``slots[r]`` (positions[r] without slots; -1: a padding row) of sequence
    ``seq_ids[r]`` (0 without) and returns q [rows, Hq, hd] rotated (``q_out``, made when
    not given; ``q_out=q`` in place; None without q). Without a table nothing is
    rotated."""
    if stream is not None and q is not None and q_out is None:
        q_out = _like(q, stream)
    if table is None:
        tdata, max_pos, rotary_dim = None, 0, 0
    else:
        tdata, max_pos, rotary_dim = table.data, table.max_pos, table.head_dim
    return _lib.serving_ops().paged_kv_append(q, k, v, positions, slots, seq_ids, cache.k_pages, cache.v_pages, cache.page_table,
                                              tdata, max_pos, rotary_dim, interleaved, q_out, _word(status), _handle(stream))


def paged_tree_attention_workspace(q: torch.Tensor, cache: PagedKV, batch: int, max_ctx: int, max_tree: int,
                                   stream=None) -> torch.Tensor:
    """Device scratch for paged_tree_attention calls of these sizes (q's rows, batch and
    bounds). Calls that overlap on the GPU need one each."""
    if q.dim() != 3:
        raise _invalid("q must be [rows, heads, head_dim]")
    _dev(q)
    n = ctypes.c_size_t()
    with torch.cuda.device(cache.device):
        check(load().bm_paged_tree_attention_workspace_size(q.shape[0], batch, q.shape[1], cache.num_kv_heads,
                                                            cache.head_dim, max_ctx, max_tree, ctypes.byref(n)))
    return _empty((n.value,), torch.uint8, cache.device, stream)


def paged_tree_attention(q: torch.Tensor, cache: PagedKV, ctx_lens: torch.Tensor, q_starts: torch.Tensor,
                         max_ctx: int, max_tree: int, tree_mask: Optional[torch.Tensor] = None,
                         seq_ids: Optional[torch.Tensor] = None, scale: float = 0.0,
                         out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                         status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """Attention of each sequence's drafted tokens over its cached context and over the
    drafted tokens that they see. q [rows, Hq, hd] holds sequence b's rows
    q_starts[b]:q_starts[b + 1]; its context is the cache slots before ctx_lens[b], its
    drafted tokens' K and V are in the slots behind (paged_kv_append). Bit j % 64 of
    ``tree_mask`` (int64 [rows, words])[row, j // 64] lets the row see drafted token j;
    without a mask row i sees j <= i (a prompt's chunk; with one row, decode attention).
    max_ctx and max_tree bound ctx_lens and a sequence's rows. Rows outside every
    sequence are left as they were in ``out``. ``workspace``:
    paged_tree_attention_workspace's, made for the call when None."""
    if workspace is None:
        workspace = paged_tree_attention_workspace(q, cache, ctx_lens.numel(), max_ctx, max_tree, stream)
    if stream is not None and out is None:
        out = _like(q, stream)
    return _lib.serving_ops().paged_tree_attention(q, cache.k_pages, cache.v_pages, cache.page_table, ctx_lens, q_starts,
                                                   max_ctx, max_tree, tree_mask, seq_ids, scale, out, workspace, _word(status), _handle(stream))


def qk_norm_rotary(q: Optional[torch.Tensor], k: Optional[torch.Tensor], q_weight: Optional[torch.Tensor],
                   k_weight: Optional[torch.Tensor], positions, table: RopeTable, eps: float = 1e-5,
                   interleaved: bool = False, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                   status: Optional[DeviceStatus] = None, stream=None):
    """rotary of heads that are normed first: every head x of q and k becomes x * rsqrt(mean(x^2) +
    eps) * its weight [head_dim] and is rotated, in one pass, with one rounding. Everything else as
    rotary has it; either of q and k may be None, with its weight. head_dim <= 256."""
    if table is None:
        raise _invalid("qk_norm_rotary needs a table")
    if positions is None:
        raise _invalid("qk_norm_rotary needs positions")
    if stream is not None:
        q_out = _like(q, stream) if q is not None and q_out is None else q_out
        k_out = _like(k, stream) if k is not None and k_out is None else k_out
    pos, pos0 = (None, positions) if isinstance(positions, int) else (positions, 0)
    return _lib.serving_ops().qk_norm_rotary(q, k, q_weight, k_weight, eps, pos, pos0, table.data, table.max_pos, table.head_dim,
                                             interleaved, q_out, k_out, _word(status), _handle(stream))


class PagedKV8:
    """A paged KV cache in 8 bits over the caller's tensors: k_pages and v_pages float8_e4m3fn
    [num_pages, Hkv, page_size, hd], k_scales and v_scales float8_e8m0fnu [num_pages, Hkv,
    page_size // block] (powers of two: the value of a slot's elements is code times the scale
    of its block of slots) and page_table int32 [num_seqs, max_pages], all contiguous on one
    device; hd a multiple of 16 up to 256. Like a PagedKV's, its tensors are read by each call."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor,
                 page_table: torch.Tensor):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise _invalid("k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim]")
        if k_pages.dtype != torch.float8_e4m3fn or v_pages.dtype != torch.float8_e4m3fn:
            raise _invalid("k_pages and v_pages must be float8_e4m3fn")
        if k_pages.shape[3] % 16 or not 16 <= k_pages.shape[3] <= 256:
            raise _invalid("head_dim of an 8-bit cache must be a multiple of 16 up to 256")
        if (k_scales.dim() != 3 or k_scales.shape != v_scales.shape or k_scales.shape[:2] != k_pages.shape[:2]
                or k_scales.shape[2] == 0 or k_pages.shape[2] % k_scales.shape[2]):
            raise _invalid("k_scales and v_scales must be [num_pages, kv_heads, page_size / block]")
        if k_scales.dtype != torch.float8_e8m0fnu or v_scales.dtype != torch.float8_e8m0fnu:
            raise _invalid("k_scales and v_scales must be float8_e8m0fnu")
        for t, n in ((k_pages, "k_pages"), (v_pages, "v_pages"), (k_scales, "k_scales"), (v_scales, "v_scales")):
            _dense(t, n)
            if t.device != _dev(k_pages):
                raise _invalid("tensors must share device")
        if page_table.dim() != 2:
            raise _invalid("page_table must be [num_seqs, max_pages]")
        if page_table.dtype != torch.int32 or not page_table.is_contiguous() or page_table.device != _dev(k_pages):
            raise _invalid("page_table must be a contiguous int32 tensor on the pages' device")
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self.page_table = page_table

    num_pages = property(lambda self: self.k_pages.shape[0])
    num_kv_heads = property(lambda self: self.k_pages.shape[1])
    page_size = property(lambda self: self.k_pages.shape[2])
    block = property(lambda self: self.k_pages.shape[2] // self.k_scales.shape[2])
    head_dim = property(lambda self: self.k_pages.shape[3])
    num_seqs = property(lambda self: self.page_table.shape[0])
    max_pages = property(lambda self: self.page_table.shape[1])
    device = property(lambda self: self.k_pages.device)


def paged_kv8_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cache: PagedKV8, ctx_lens: torch.Tensor,
                     q_starts: torch.Tensor, max_tokens: int, positions: Optional[torch.Tensor] = None,
                     table: Optional[RopeTable] = None, q_weight: Optional[torch.Tensor] = None,
                     k_weight: Optional[torch.Tensor] = None, eps: float = 1e-5, seq_ids: Optional[torch.Tensor] = None,
                     interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                     status: Optional[DeviceStatus] = None, stream=None) -> Optional[torch.Tensor]:
    """Appends sequence b's rows q_starts[b]:q_starts[b + 1] of k and v [rows, Hkv, hd] (at most
    max_tokens) to its slots from ctx_lens[b] on, quantised, and returns q [rows, Hq, hd]
    (``q_out``, made when not given; ``q_out=q`` in place; None without q): q and k normed with
    q_weight and k_weight [hd] (None: not) and rotated by ``table`` (None: not) at ``positions``
    (None: their slots). A block's scale is the power of two that its largest value needs; it
    grows, and earlier codes of the block with it, where new rows are larger, and is set afresh
    where a call writes the block's first slot. ctx_lens, q_starts and seq_ids are
    paged_kv8_tree_attention's. Rows of ``q_out`` outside every sequence are left as they were.
    A call must not name a sequence twice."""
    if stream is not None and q is not None and q_out is None:
        q_out = _like(q, stream)
    if table is None:
        tdata, max_pos, rotary_dim = None, 0, 0
    else:
        tdata, max_pos, rotary_dim = table.data, table.max_pos, table.head_dim
    return _lib.serving_ops().paged_kv8_append(q, k, v, cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, cache.page_table,
                                               ctx_lens, q_starts, max_tokens, positions, tdata, max_pos, rotary_dim, q_weight,
                                               k_weight, eps, seq_ids, interleaved, q_out, _word(status), _handle(stream))


def paged_kv8_read(cache: PagedKV8, first: torch.Tensor, starts: torch.Tensor, rows: int, max_rows: int,
                   dtype: torch.dtype = torch.bfloat16, seq_ids: Optional[torch.Tensor] = None,
                   k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None,
                   status: Optional[DeviceStatus] = None, stream=None):
    """Cached slots as dense values: rows starts[b]:starts[b + 1] (at most max_rows) of k and v
    [rows, Hkv, hd] are sequence b's slots from first[b] on; exact in bf16 and fp32. Returns
    (k_out, v_out), made when not given, of ``dtype``; rows outside every sequence are left as
    they were."""
    shape = (rows, cache.num_kv_heads, cache.head_dim)
    if rows < 0:
        raise _invalid("rows must be >= 0")
    for out in (k_out, v_out):
        if out is not None and out.shape != shape:
            raise _invalid("k_out and v_out must be [rows, kv_heads, head_dim]")
    given = k_out if k_out is not None else v_out
    if given is not None:
        dtype = given.dtype
    if k_out is None:
        k_out = _empty(shape, dtype, cache.device, stream)
    if v_out is None:
        v_out = _empty(shape, dtype, cache.device, stream)
    return _lib.serving_ops().paged_kv8_read(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, cache.page_table, first,
                                             starts, max_rows, seq_ids, k_out, v_out, _word(status), _handle(stream))


def paged_kv8_tree_attention_workspace(q: torch.Tensor, cache: PagedKV8, batch: int, max_ctx: int, max_tree: int,
                                       stream=None) -> torch.Tensor:
    """Device scratch for paged_kv8_tree_attention calls of these sizes (q's rows, batch and
    bounds). Calls that overlap on the GPU need one each."""
    if q.dim() != 3:
        raise _invalid("q must be [rows, heads, head_dim]")
    _dev(q)
    n = ctypes.c_size_t()
    with torch.cuda.device(cache.device):
        check(load().bm_paged_kv8_tree_attention_workspace_size(q.shape[0], batch, q.shape[1], cache.num_kv_heads,
                                                                cache.head_dim, max_ctx, max_tree, ctypes.byref(n)))
    return _empty((n.value,), torch.uint8, cache.device, stream)


def paged_kv8_tree_attention(q: torch.Tensor, cache: PagedKV8, ctx_lens: torch.Tensor, q_starts: torch.Tensor,
                             max_ctx: int, max_tree: int, tree_mask: Optional[torch.Tensor] = None,
                             seq_ids: Optional[torch.Tensor] = None, scale: float = 0.0,
                             out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                             status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """paged_tree_attention over an 8-bit cache: the same arguments and rules, with q and out of
    bf16 or fp32. ``workspace``: paged_kv8_tree_attention_workspace's, made for the call when None."""
    if workspace is None:
        workspace = paged_kv8_tree_attention_workspace(q, cache, ctx_lens.numel(), max_ctx, max_tree, stream)
    if stream is not None and out is None:
        out = _like(q, stream)
    return _lib.serving_ops().paged_kv8_tree_attention(q, cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales,
                                                       cache.page_table, ctx_lens, q_starts, max_ctx, max_tree, tree_mask, seq_ids,
                                                       scale, out, workspace, _word(status), _handle(stream))


def sample(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           status: Optional[DeviceStatus] = None, stream=None) -> torch.Tensor:
    """One token per row of logits [rows, vocab] from uniforms [rows] in [0, 1):
    temperature, then top-k, top-p and min-p (each a tensor of one entry per row, or None:
    off), then the first index whose running weight exceeds its uniform's share. Ties
    go to the lowest index; temperature 0 takes the largest logit; a row without any
    weight gives -1. Returns int32 [rows]."""
    if stream is not None and out is None:
        out = _empty((logits.shape[0],), torch.int32, _dev(logits), stream)
    return _lib.serving_ops().sample(logits, uniforms, temperature, top_k, top_p, min_p, out, _word(status), _handle(stream))


# --------------------------------------------------------------------------
# The reference's launch API (single token, fp32), include/kernels.cuh
# --------------------------------------------------------------------------

def layer_step(ids: torch.Tensor, embed: torch.Tensor, hidden: torch.Tensor, attn_out: torch.Tensor,
               w_attn: torch.Tensor, y_attn: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
               positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, ffn_out: torch.Tensor,
               w_ffn: torch.Tensor, y_ffn: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, act: torch.Tensor,
               eps: float = 1e-5, table: Optional[RopeTable] = None, theta: float = 10000.0,
               seq_ids: Optional[torch.Tensor] = None, status: Optional[DeviceStatus] = None, stream=None) -> None:
    """One layer step (bm_layer_step): hidden = embed[ids] + attn_out, y_attn =
    rmsnorm(hidden) * w_attn, RoPE on q (in place) and k into k_cache with v into
    v_cache, hidden += ffn_out, y_ffn = rmsnorm(hidden) * w_ffn, act = silu(gate)
    * up. One launch for batches of at most 512 tokens, five otherwise."""
    rows, dim = hidden.shape
    for t, n in ((embed, "embed"), (hidden, "hidden"), (attn_out, "attn_out"), (w_attn, "w_attn"),
                 (y_attn, "y_attn"), (q, "q"), (k, "k"), (v, "v"), (k_cache, "k_cache"), (v_cache, "v_cache"),
                 (ffn_out, "ffn_out"), (w_ffn, "w_ffn"), (y_ffn, "y_ffn"), (gate, "gate"), (up, "up"), (act, "act")):
        _dense(t, n)
    _same(hidden, embed, attn_out, w_attn, y_attn, q, k, v, k_cache, v_cache, ffn_out, w_ffn, y_ffn, gate, up, act)
    _i32(ids, "ids")
    _i32(positions, "positions")
    _i32(seq_ids, "seq_ids")
    ffn = gate.shape[-1]
    shapes_ok = (attn_out.shape == hidden.shape == y_attn.shape == ffn_out.shape == y_ffn.shape
                 and embed.shape[1] == dim and w_attn.numel() == dim and w_ffn.numel() == dim
                 and gate.shape == up.shape == act.shape == (rows, ffn) and ids.numel() == rows
                 and positions.numel() == rows and q.shape[0] == rows and k.shape == v.shape
                 and k.shape[0] == rows and k_cache.shape == v_cache.shape and k_cache.shape[1] == k.shape[1]
                 and (seq_ids is None or seq_ids.numel() == rows))
    if not shapes_ok:
        raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "layer step tensor shapes disagree")
    c = _lib.LayerStepC()
    c.rows, c.dim, c.ffn, c.vocab = rows, dim, ffn, embed.shape[0]
    c.num_q_heads, c.num_kv_heads, c.head_dim = q.shape[1], k.shape[1], q.shape[2]
    c.max_seq, c.num_seqs, c.eps, c.theta = k_cache.shape[2], k_cache.shape[0], eps, theta
    c.ids, c.embed, c.hidden, c.attn_out, c.w_attn, c.y_attn = (_ptr(ids), _ptr(embed), _ptr(hidden), _ptr(attn_out),
                                                                _ptr(w_attn), _ptr(y_attn))
    c.q, c.k, c.v, c.positions, c.seq_ids = _ptr(q), _ptr(k), _ptr(v), _ptr(positions), _ptr(seq_ids)
    c.k_cache, c.v_cache = _ptr(k_cache), _ptr(v_cache)
    c.rope_table = None if table is None else table.ptr
    c.rope_table_len = 0 if table is None else table.max_pos
    c.ffn_out, c.w_ffn, c.y_ffn, c.gate, c.up, c.act = (_ptr(ffn_out), _ptr(w_ffn), _ptr(y_ffn), _ptr(gate),
                                                        _ptr(up), _ptr(act))
    with torch.cuda.device(_dev(hidden)):
        check(load().bm_layer_step(ctypes.byref(c), bm_dtype(hidden), None if status is None else status.ptr,
                                   _stream(hidden.device, stream)))


def _stream_arg(stream) -> int:
    if stream is None or stream == 0:
        return 0
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def launch_rms_norm(out: torch.Tensor, inp: torch.Tensor, weight: torch.Tensor, size: int, eps: float = 1e-5,
                    stream=0) -> None:
    """include/kernels.cuh:9 — one vector of ``size`` floats; out may be inp."""
    with torch.cuda.device(_dev(inp)):
        check(load().bm_rmsnorm(_ptr(out), _ptr(inp), _ptr(weight), 1, size, eps, size, size, _lib.BM_F32,
                                _stream_arg(stream)))


def launch_rope(q: torch.Tensor, k: torch.Tensor, seq_pos: int, head_dim: int, num_heads: int, num_kv_heads: int,
                theta: float = 10000.0, stream=0) -> None:
    """include/kernels.cuh:15 — rotates one token's q and k in place."""
    with torch.cuda.device(_dev(q)):
        check(load().bm_rope(_ptr(q), _ptr(k), None, seq_pos, None, 0, float(theta), 1, num_heads, num_kv_heads,
                             head_dim, _lib.BM_F32, None, _stream_arg(stream)))


def launch_gemm(c: torch.Tensor, a: torch.Tensor, b: torch.Tensor, m: int, n: int, k: int, stream=0) -> None:
    """include/kernels.cuh:20 — c[m][n] = a[m][k] b[k][n], fp32."""
    with torch.cuda.device(_dev(a)):
        check(load().bm_gemm(_ptr(c), _ptr(a), _ptr(b), m, n, k, _lib.BM_F32, None, _stream_arg(stream)))


def launch_softmax_batch(x: torch.Tensor, size: int, num_vectors: int, stride: int, stream=0) -> None:
    """include/kernels.cuh:26 — softmax in place over num_vectors vectors `stride` apart."""
    with torch.cuda.device(_dev(x)):
        check(load().bm_softmax(_ptr(x), size, num_vectors, stride, _lib.BM_F32, _stream_arg(stream)))


def launch_softmax(x: torch.Tensor, size: int, stream=0) -> None:
    """include/kernels.cuh:23 — softmax in place over one vector."""
    launch_softmax_batch(x, size, 1, size, stream)


def launch_swiglu(out: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, size: int, stream=0) -> None:
    """include/kernels.cuh:29 — out = silu(gate) * up."""
    with torch.cuda.device(_dev(gate)):
        check(load().bm_swiglu(_ptr(out), _ptr(gate), _ptr(up), size, _lib.BM_F32, _stream_arg(stream)))


def launch_add(out: torch.Tensor, a: torch.Tensor, b: torch.Tensor, size: int, stream=0) -> None:
    """include/kernels.cuh:32 — out = a + b; out may alias a or b."""
    with torch.cuda.device(_dev(a)):
        check(load().bm_add(_ptr(out), _ptr(a), _ptr(b), size, _lib.BM_F32, _stream_arg(stream)))


def launch_kv_store(cache: torch.Tensor, src: torch.Tensor, seq_pos: int, num_heads: int, head_dim: int,
                    max_seq_len: int, stream=0) -> None:
    """include/kernels.cuh:36 — cache [H][max_seq][hd] at seq_pos = src [H][hd]."""
    with torch.cuda.device(_dev(src)):
        check(load().bm_kv_store(_ptr(cache), _ptr(src), None, seq_pos, None, 1, num_heads, head_dim, max_seq_len,
                                 1, _lib.BM_F32, None, _stream_arg(stream)))


# --------------------------------------------------------------------------
# Batch-aware KV cache (bm_kv_cache_*)
# --------------------------------------------------------------------------

class KVCache:
    """Per-layer K/V caches [num_seqs][kv_heads][max_seq][head_dim] with one length
    per sequence (the reference's KVCache, include/kv_cache.h:10-40, keeps one
    position for the whole cache). Create it with the target device current."""

    def __init__(self, num_layers: int, num_seqs: int, num_kv_heads: int, max_seq: int, head_dim: int,
                 max_tokens: int, dtype: torch.dtype = torch.bfloat16, device=None):
        self.dtype = dtype
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.shape = (num_seqs, num_kv_heads, max_seq, head_dim)
        self.num_layers = num_layers
        handle = ctypes.c_void_p()
        with torch.cuda.device(self.device):
            check(load().bm_kv_cache_create(num_layers, num_seqs, num_kv_heads, max_seq, head_dim, max_tokens,
                                            _DTYPES[dtype], ctypes.byref(handle)))
        self._h = handle

    def close(self) -> None:
        if self._h:
            with torch.cuda.device(self.device):
                check(load().bm_kv_cache_destroy(self._h))
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass

    def layer_ptrs(self, layer: int):
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        check(load().bm_kv_cache_layer(self._h, layer, ctypes.byref(k), ctypes.byref(v)))
        return k.value, v.value

    def seq_len(self, seq: int) -> int:
        n = ctypes.c_int32()
        check(load().bm_kv_cache_seq_len(self._h, seq, ctypes.byref(n)))
        return n.value

    def reset(self, seq: int = -1) -> None:
        check(load().bm_kv_cache_reset(self._h, seq))

    def append(self, seq_ids, stream=None):
        """Assigns the next position of its sequence to each new token (seq_ids: host
        ints); returns device pointers (positions, seq_ids) for rope_kv_store."""
        import numpy as np

        ids = np.ascontiguousarray(np.asarray(seq_ids, dtype=np.int32))
        pos_p, seq_p = ctypes.c_void_p(), ctypes.c_void_p()
        with torch.cuda.device(self.device):
            check(load().bm_kv_cache_append(self._h, ids.ctypes.data if ids.size else None, ids.size,
                                            ctypes.byref(pos_p), ctypes.byref(seq_p),
                                            _stream(self.device, stream)))
        return pos_p.value, seq_p.value, ids.size

    def rope_kv_store(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, appended,
                      table: Optional[RopeTable] = None, theta: float = 10000.0,
                      status: Optional[DeviceStatus] = None, stream=None) -> None:
        """bm_rope_kv_store into `layer` for the tokens of the last append()."""
        pos_p, seq_p, rows = appended
        kc, vc = self.layer_ptrs(layer)
        num_seqs, hkv, max_seq, hd = self.shape
        for t, n in ((q, "q"), (k, "k"), (v, "v")):
            _dense(t, n)
        _same(q, k, v)
        if q.dtype != self.dtype or q.shape[0] != rows or k.shape[1] != hkv or q.shape[2] != hd:
            raise BMError(_lib.BM_ERR_INVALID_ARGUMENT, "q/k/v do not match the cache or the appended tokens")
        with torch.cuda.device(_dev(q)):
            check(load().bm_rope_kv_store(_ptr(q), _ptr(k), _ptr(v), pos_p, 0, seq_p, kc, vc,
                                          table.ptr if table else None, table.max_pos if table else 0, theta,
                                          rows, q.shape[1], hkv, hd, max_seq, num_seqs, bm_dtype(q),
                                          status.ptr if status else None, _stream(q.device, stream)))

    def views(self, layer: int):
        """Layer `layer`'s K and V caches as torch tensors viewing the cache's
        memory (no copy; valid while the cache lives)."""
        typestr = "<f4" if self.dtype == torch.float32 else "<i2"
        out = []
        for p in self.layer_ptrs(layer):
            arr = _DeviceArray(p, self.shape, typestr)
            t = torch.as_tensor(arr, device=self.device)
            out.append(t if self.dtype == torch.float32 else t.view(torch.bfloat16))
        return out


class _DeviceArray:
    """A raw device allocation described by __cuda_array_interface__ (v3)."""

    def __init__(self, ptr: int, shape, typestr: str):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3, "strides": None}
