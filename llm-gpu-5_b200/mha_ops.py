"""Launch wrappers over the C ABI, in the role core/mha_ops.py plays for the reference.

Each wrapper takes torch CUDA tensors (or raw device addresses), checks shapes on the host,
and launches on the current torch stream.  All compute is in libattn_b200.so.

The reference's launch constants (core/mha_ops.py:22-23) are kept for callers that read them;
the kernels here choose their own tiling.
"""

from __future__ import annotations

import functools
import math
import operator

import torch

from ._lib import ATTN_ACT_GELU, ATTN_ACT_GELU_BWD, ATTN_ACT_NONE, ATTN_BF16, ATTN_F32, ATTN_TF32, AttnError, call, last_error, lib  # noqa: F401

THREADS_PER_BLOCK = 256
SOFTMAX_BLOCK_THREADS = 64

_DT = {torch.float32: ATTN_F32, torch.bfloat16: ATTN_BF16}


def dtype_code(t) -> int:
    """Library code of an operand type: torch.float32, torch.bfloat16, or "tf32" (float32 storage
    multiplied on the tensor cores as tf32)."""
    if isinstance(t, str) and t == "tf32":
        return ATTN_TF32
    try:
        return _DT[t]
    except KeyError:
        raise TypeError(f"unsupported dtype {t}; expected float32, bfloat16 or 'tf32'") from None


def _stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(x) -> int:
    """Device address of a torch tensor, a DeviceBuffer, a pycuda DeviceAllocation or an int."""
    if isinstance(x, torch.Tensor):
        if not x.is_cuda:
            raise TypeError("expected a CUDA tensor")
        return x.data_ptr()
    if hasattr(x, "data_ptr"):
        return int(x.data_ptr())
    return int(x)


class HeadView:
    """Element strides of an attention operand: element (b, t, h, d) at base[b*sb + t*st + h*sh + d]."""

    __slots__ = ("base", "sb", "st", "sh")

    def __init__(self, base: int, sb: int, st: int, sh: int):
        self.base, self.sb, self.st, self.sh = int(base), int(sb), int(st), int(sh)

    @staticmethod
    def tokens(base: int, T: int, ld: int, D: int) -> "HeadView":
        """Token layout [B*T, ld] with head h at column offset h*D (the fused projection layout)."""
        return HeadView(base, T * ld, ld, D)

    @staticmethod
    def heads(base: int, NH: int, T: int, D: int) -> "HeadView":
        """The reference's split layout [B*NH, T, D] (split_heads_kernel output)."""
        return HeadView(base, NH * T * D, D, T * D)


def attention_forward(q: HeadView, k: HeadView, v: HeadView, o: HeadView, lse: torch.Tensor,
                      B: int, NH: int, T: int, D: int, scale: float, dtype: torch.dtype):
    """Causal attention forward; q/k/v share strides.  lse: float32 [B, NH, T]."""
    assert (k.sb, k.st, k.sh) == (q.sb, q.st, q.sh) == (v.sb, v.st, v.sh)
    assert lse.dtype == torch.float32 and lse.numel() >= B * NH * T
    call("attn_fwd", q.base, k.base, v.base, o.base, lse.data_ptr(), B, NH, T, D,
         q.sb, q.st, q.sh, o.sb, o.st, o.sh, float(scale), dtype_code(dtype), _stream())


def attention_backward(q: HeadView, k: HeadView, v: HeadView, o: HeadView, do: HeadView,
                       lse: torch.Tensor, dq: HeadView, dk: HeadView, dv: HeadView,
                       B: int, NH: int, T: int, D: int, scale: float, dtype: torch.dtype,
                       workspace: torch.Tensor | None = None):
    """Causal attention backward.  dq/dk/dv use q's strides, do uses o's."""
    assert (dq.sb, dq.st, dq.sh) == (q.sb, q.st, q.sh) == (dk.sb, dk.st, dk.sh) == (dv.sb, dv.st, dv.sh)
    assert (do.sb, do.st, do.sh) == (o.sb, o.st, o.sh)
    code = dtype_code(dtype)
    need = lib.attn_bwd_workspace_size(B, NH, T, D, code)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
    call("attn_bwd", q.base, k.base, v.base, o.base, do.base, lse.data_ptr(), dq.base, dk.base,
         dv.base, workspace.data_ptr(), workspace.numel() * workspace.element_size(), B, NH, T, D,
         q.sb, q.st, q.sh, o.sb, o.st, o.sh, float(scale), code, _stream())


def attention_probs(q: HeadView, k: HeadView, lse: torch.Tensor, B, NH, T, D, scale, dtype):
    """Rebuild the [B, NH, T, T] probabilities from lse (debug/test accessor)."""
    out = torch.empty((B, NH, T, T), dtype=torch.float32, device="cuda")
    call("attn_probs", q.base, k.base, lse.data_ptr(), out.data_ptr(), B, NH, T, D, q.sb, q.st, q.sh,
         float(scale), dtype_code(dtype), _stream())
    return out


def decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scale: float | None = None,
           out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None):
    """Single-query decode: q [B, NH, D], caches [B, L, NH, D] (token layout) -> out [B, NH, D]."""
    B, NH, D = q.shape
    L = k_cache.shape[1]
    assert k_cache.shape == v_cache.shape == (B, L, NH, D)
    assert q.dtype == k_cache.dtype == v_cache.dtype
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    # q and out are addressed with the same (b, h) strides
    assert out.shape == q.shape and out.dtype == q.dtype and out.stride() == q.stride(), \
        "decode: q and out must have the same shape, dtype and strides"
    need = lib.attn_decode_workspace_size(B, NH, L, D)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    qs = q.stride()
    ks = k_cache.stride()
    assert k_cache.stride() == v_cache.stride() and ks[3] == 1 and qs[2] == 1
    call("attn_decode", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
         lse.data_ptr() if lse is not None else None, B, NH, L, D, qs[0], qs[1], ks[0], ks[1], ks[2],
         float(scale), dtype_code(q.dtype), workspace.data_ptr(),
         workspace.numel() * workspace.element_size(), _stream())
    return out


# ---------------------------------------------------------------- 4-bit key/value cache
# codes: uint8 [2, B, NH, cap, D/2]; params: float16 [2, B, NH, cap, D/min(D, 64), 2], index 0 keys and
# 1 values (the format is described in include/attn_b200.h).  Views along the sequence and head axes
# are taken as they are; both arrays must be the same view.

KV4_HEAD_DIMS = (16, 32, 64, 128)
KV4_ROWS = 16  # capacity and strides are multiples of this many rows


def kv4_groups(D: int) -> int:
    """Scale pairs per cached row of D values."""
    return D // min(D, 64)


def kv4_empty(B: int, NH: int, capacity: int, D: int, device="cuda"):
    """Uninitialised (codes, params) of a cache of ``capacity`` rows (rounded up to a multiple of 16)
    per sequence and head."""
    if D not in KV4_HEAD_DIMS:
        raise ValueError(f"the 4-bit cache takes head_dim 16, 32, 64 or 128, got {D}")
    cap = (capacity + KV4_ROWS - 1) // KV4_ROWS * KV4_ROWS
    return (torch.empty((2, B, NH, cap, D // 2), dtype=torch.uint8, device=device),
            torch.empty((2, B, NH, cap, kv4_groups(D), 2), dtype=torch.float16, device=device))


# The checks below run once per call of operators whose kernels take a few microseconds for a token: they
# unpack shapes and strides once and compare dtypes by identity.
_U8, _F16 = torch.uint8, torch.float16
_OF = {code: dtype for dtype, code in _DT.items()}


def _kv4_view(codes: torch.Tensor, params: torch.Tensor):
    """(B, NH, cap, D, strides in rows) of a cache's two arrays, checked."""
    if codes.dtype is not _U8 or params.dtype is not _F16:
        raise TypeError(f"4-bit cache: codes must be uint8 and params float16, got {codes.dtype} and {params.dtype}")
    shape = codes.shape
    if len(shape) != 5 or params.device != codes.device or not codes.is_cuda:
        raise ValueError("4-bit cache: expected CUDA codes [2, B, NH, cap, D/2] and params [2, B, NH, cap, groups, 2]")
    two, B, NH, cap, half = shape
    if half not in (8, 16, 32, 64):
        raise ValueError(f"the 4-bit cache takes head_dim 16, 32, 64 or 128, got {2 * half}")
    G = 2 if half == 64 else 1
    if two != 2 or params.shape != (2, B, NH, cap, G, 2):
        raise ValueError(f"4-bit cache: codes {tuple(shape)} and params {tuple(params.shape)} do not match")
    c0, c1, c2, c3, c4 = codes.stride()
    p0, p1, p2, p3, p4, p5 = params.stride()
    sh = c2 // half if NH > 1 else cap
    sb = c1 // half if B > 1 else NH * cap
    si = c0 // half
    if c3 != half or c4 != 1 or p3 != 2 * G or p4 != 2 and G > 1 or p5 != 1 or si * half != c0 or p0 != si * 2 * G \
            or (B > 1 and (sb * half != c1 or p1 != sb * 2 * G)) or (NH > 1 and (sh * half != c2 or p2 != sh * 2 * G)):
        raise ValueError("4-bit cache: rows must be contiguous and both arrays the same view")
    return B, NH, cap, 2 * half, si, sb, sh


def _kv4_marks(name, t, dtype, B, NH, rows, device):
    """(address, sequence stride, head stride) of a [B, NH, >= rows] array beside the cache."""
    if t is None:
        return None, 0, 0
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[0] != B or shape[1] != NH or shape[2] < rows or t.device != device:
        raise ValueError(f"{name}: expected [{B}, {NH}, >= {rows}] on {device}, got {tuple(shape)} on {t.device}")
    sb, sh, sl = t.stride()
    if sl != 1 and shape[2] > 1:
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr(), sb, sh


def _int32(name, x):
    """x as an int that C takes whole: ctypes drops the bits above an int's 32."""
    x = operator.index(x)
    if not -0x80000000 <= x <= 0x7fffffff:
        raise ValueError(f"{name}: {x} does not fit 32 bits")
    return x


def _per_sequence(name, x, B, device):
    """(device address or None, int to add) of an int or an int32 tensor of one entry per sequence."""
    if not isinstance(x, torch.Tensor):
        return None, _int32(name, x)
    if x.dtype != torch.int32:
        raise TypeError(f"{name}: expected an int or int32, got {x.dtype}")
    if x.shape != (B,) or x.device != device or not x.is_contiguous():
        raise ValueError(f"{name}: expected {B} contiguous entries on {device}, got {tuple(x.shape)} on {x.device}")
    return x.data_ptr(), 0


def _row_counts(name, x, B, device):
    """Device address of an int32 tensor of one entry per sequence, or None."""
    if x is None:
        return None
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: expected an int32 tensor of one entry per sequence, got {type(x).__name__}")
    return _per_sequence(name, x, B, device)[0]


def _public_raw_stream(index):
    return torch.cuda.current_stream(index).cuda_stream


# The current stream's handle without building a torch.cuda.Stream: 0.1 against 3.2 us of a call that
# takes 10 in all.  Neither name is one that torch promises to keep; its public calls stand in for them.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_raw_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _other_device(device):
    """Make the tensors' device the current one where it is not; what was current, to go back to, or None."""
    index = _current_device()
    if device.index == index:
        return None
    torch.cuda.set_device(device)
    return index


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(name, *sizes):
    """What a *_workspace_size function answers for these sizes (and current device)."""
    return getattr(lib, name)(*sizes[1:])


def _scratch(workspace, need: int, like):
    """(tensor to keep alive, address, bytes) of a workspace: the caller's, or a new one beside ``like``."""
    if workspace is None:
        if not need:
            return None, None, 0
        workspace = like.new_empty(need, dtype=torch.uint8)
        return workspace, workspace.data_ptr(), need
    if workspace.device != like.device or not workspace.is_contiguous():
        raise ValueError(f"workspace: expected a contiguous tensor on {like.device}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _token_rows(name, x, B, NH, D, device):
    """Strides of a [B, T, NH, D] operand with contiguous rows."""
    shape = x.shape
    if len(shape) != 4 or shape[0] != B or shape[2] != NH or shape[3] != D or x.device != device:
        raise ValueError(f"{name}: expected [{B}, T, {NH}, {D}] on {device}, got {tuple(shape)} on {x.device}")
    st = x.stride()
    if st[3] != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    return st


def kv4_store(k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, pos, counts=None,
              weights=None, positions=None, seen=None):
    """Quantise keys and values [B, T, NH, D] (float32 or bfloat16, any strides with contiguous rows)
    into slots pos .. pos+T-1 of a 4-bit cache.

    ``pos`` is an int or an int32 tensor [B]; ``counts`` (int32 [B]) leaves the rows of shorter
    sequences as they were.  ``weights`` (float32) and ``positions`` (int32), [B, NH, >= capacity], get 0 and
    the token positions seen, seen+1, ... (``seen``: int or int32 [B], by default ``pos``)."""
    B, NH, cap, D, si, sb, sh = _kv4_view(codes, params)
    dev = codes.device
    ks, vs = _token_rows("k", k, B, NH, D, dev), _token_rows("v", v, B, NH, D, dev)
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"kv4_store: k and v differ: {tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
    T = k.shape[1]
    if T == 0 or B == 0:
        return
    code = dtype_code(k.dtype)
    _int32("T", T)
    wp, wsb, wsh = _kv4_marks("weights", weights, torch.float32, B, NH, cap, dev)
    pp, psb, psh = _kv4_marks("positions", positions, torch.int32, B, NH, cap, dev)
    if wp is not None and pp is not None and (wsb, wsh) != (psb, psh):
        raise ValueError("kv4_store: weights and positions must have the same strides")
    if wp is None:
        wsb, wsh = psb, psh
    starts, start = _per_sequence("pos", pos, B, dev)
    seen_p, seen0 = _per_sequence("seen", pos if seen is None else seen, B, dev)
    if pp is not None:
        _int32("positions", seen0 + T - 1)
    counts_p = _row_counts("counts", counts, B, dev)
    before = _other_device(dev)
    try:
        rc = lib.attn_kv4_store(k.data_ptr(), v.data_ptr(), code, B, T, NH, D, ks[0], ks[1], ks[2],
                                vs[0], vs[1], vs[2], codes.data_ptr(), params.data_ptr(), si, sb, sh, cap, starts, start, counts_p, wp, pp,
                                wsb, wsh, seen_p, seen0, _raw_stream(dev.index))
    finally:
        if before is not None:
            torch.cuda.set_device(before)
    if rc:
        raise AttnError("attn_kv4_store", rc, last_error())


def kv4_load(codes: torch.Tensor, params: torch.Tensor, pos, T: int, dtype: torch.dtype = torch.float32, counts=None):
    """The numbers held in slots pos .. pos+T-1 of a 4-bit cache: (k, v), each [B, T, NH, D] of
    ``dtype``; zeros for the rows from ``counts`` on and for slots outside the cache."""
    B, NH, cap, D, si, sb, sh = _kv4_view(codes, params)
    dev = codes.device
    _int32("T", T)
    code = dtype_code(dtype)
    k = codes.new_empty((B, T, NH, D), dtype=dtype)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    starts, start = _per_sequence("pos", pos, B, dev)
    counts_p = _row_counts("counts", counts, B, dev)
    before = _other_device(dev)
    try:
        rc = lib.attn_kv4_load(codes.data_ptr(), params.data_ptr(), si, sb, sh, cap, B, T, NH, D, starts, start,
                               counts_p, k.data_ptr(), v.data_ptr(), code, T * NH * D, NH * D, D, _raw_stream(dev.index))
    finally:
        if before is not None:
            torch.cuda.set_device(before)
    if rc:
        raise AttnError("attn_kv4_load", rc, last_error())
    return k, v


def kv4_decode(q: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, length: int, lengths=None,
               scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
               weights: torch.Tensor | None = None, weights_out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None):
    """Single-query decode over a 4-bit cache: q [B, NH, D] -> out [B, NH, D] of q's dtype.

    The cache's heads are shared by NH / (its heads) consecutive query heads.  Every sequence
    attends over its first ``length`` rows, or ``lengths[b]`` (int32 [B], at most ``length``; none
    gives zeros and lse -inf).  With ``weights`` (float32 [B, cached heads, >= length]) the attention
    weights are added to it, in place or into ``weights_out``; with ``weights_out`` alone they are set."""
    B, NKV, cap, D, si, sb, sh = _kv4_view(codes, params)
    dev = codes.device
    length = _int32("length", length)
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != D or q.device != dev:
        raise ValueError(f"q: expected [{B}, NH, {D}] on {dev}, got {tuple(shape)} on {q.device}")
    NH = shape[1]
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
        raise ValueError("out: must have q's shape, dtype and device")
    if lse is not None and (lse.shape != (B, NH) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != dev):
        raise ValueError(f"lse: expected contiguous float32 [{B}, {NH}] on {dev}")
    qs, os_ = q.stride(), out.stride()
    if qs[2] != 1 or os_[2] != 1:
        raise ValueError("kv4_decode: head_dim must be contiguous in q and out")
    w_in, wsb, wsh = _kv4_marks("weights", weights, torch.float32, B, NKV, length, dev)
    if weights_out is None or weights_out is weights:
        w_out = w_in
    else:
        w_out, osb, osh = _kv4_marks("weights_out", weights_out, torch.float32, B, NKV, length, dev)
        if w_in is not None and (osb, osh) != (wsb, wsh):
            raise ValueError("kv4_decode: weights and weights_out must have the same strides")
        wsb, wsh = osb, osh
    lengths_p = _row_counts("lengths", lengths, B, dev)
    code = dtype_code(q.dtype)
    if B == 0:
        return out
    before = _other_device(dev)
    try:
        need = _workspace_bytes("attn_kv4_decode_workspace_size", dev.index, B, NH, NKV, length, D, code, w_out is not None)
        workspace, ws, ws_bytes = _scratch(workspace, need, q)
        rc = lib.attn_kv4_decode(q.data_ptr(), codes.data_ptr(), params.data_ptr(), out.data_ptr(),
                                 lse.data_ptr() if lse is not None else None, B, NH, NKV, length, D, qs[0], qs[1], os_[0], os_[1], si, sb, sh,
                                 cap, lengths_p, w_in, w_out, wsb, wsh, 1.0 / math.sqrt(D) if scale is None else float(scale),
                                 code, ws, ws_bytes, _raw_stream(dev.index))
    finally:
        if before is not None:
            torch.cuda.set_device(before)
    if rc:
        raise AttnError("attn_kv4_decode", rc, last_error())
    return out


def key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, scale: float | None = None, first_query: int = 0,
                lengths=None, weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
                dtype=None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Accumulated attention weights of a causal prompt, without its T x T matrix: [B, NKV, T] float32.

    q [B, T, NH, D], k [B, T, NKV, D] (NH / NKV query heads to a key head), lse [B, NH, T] from
    ``attention_forward``: each key's attention weight summed over the queries from ``first_query``
    on (those from ``lengths[b]`` on excluded) and its query heads, added to ``weights`` when given.
    ``dtype`` "tf32" takes q and k truncated to tf32, for an lse of the tf32 forward on tensor cores (head_dim
    a multiple of 4 up to 32, aligned rows); its other layouts run in float32, and so must their weights."""
    if q.dim() != 4 or k.dim() != 4 or q.dtype != k.dtype:
        raise ValueError("key_weights: expected q [B, T, NH, D] and k [B, T, NKV, D] of one dtype")
    B, T, NH, D = q.shape
    NKV, dev = k.shape[2], q.device
    _int32("T", T)
    first_query = _int32("first_query", first_query)
    qs, ks = _token_rows("q", q, B, NH, D, dev), _token_rows("k", k, B, NKV, D, dev)
    code = dtype_code(q.dtype if dtype is None else dtype)
    if q.dtype is not (torch.float32 if code == ATTN_TF32 else _OF[code]):
        raise TypeError(f"key_weights: {dtype} does not go with operands of {q.dtype}")
    if k.shape[1] != T:
        raise ValueError(f"key_weights: q holds {T} tokens, k {k.shape[1]}")
    if lse.shape != (B, NH, T) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != dev:
        raise ValueError(f"lse: expected contiguous float32 [{B}, {NH}, {T}] on {dev}")
    if out is None:
        out = weights if weights is not None else q.new_empty((B, NKV, T), dtype=torch.float32)
    w_out, wsb, wsh = _kv4_marks("out", out, torch.float32, B, NKV, T, dev)
    w_in = None
    if weights is not None:
        w_in, isb, ish = _kv4_marks("weights", weights, torch.float32, B, NKV, T, dev)
        if (isb, ish) != (wsb, wsh):
            raise ValueError("key_weights: weights and out must have the same strides")
    lengths_p = _row_counts("lengths", lengths, B, dev)
    if B == 0 or T == 0:
        return out
    workspace, ws, ws_bytes = _scratch(workspace, _workspace_bytes("attn_key_weights_workspace_size", 0, B, NKV, T), q)
    before = _other_device(dev)
    try:
        rc = lib.attn_key_weights(q.data_ptr(), k.data_ptr(), lse.data_ptr(), w_in, w_out, B, NH, NKV, T, D,
                                  qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], wsb, wsh, first_query, lengths_p,
                                  1.0 / math.sqrt(D) if scale is None else float(scale), code,
                                  ws, ws_bytes, _raw_stream(dev.index))
    finally:
        if before is not None:
            torch.cuda.set_device(before)
    if rc:
        raise AttnError("attn_key_weights", rc, last_error())
    return out


def kv4_evict(codes: torch.Tensor, params: torch.Tensor, weights: torch.Tensor, positions, length: int, keep: int,
              recent: int = 0, seen=None, lengths=None, out=None, slots: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Keep the ``keep`` best of the ``length`` (or ``lengths[b]``) rows of every head of a 4-bit cache:
    those of the last ``recent`` of ``seen`` token positions, then those of the largest accumulated
    weight (lowest slot among equals).  Kept rows below slot ``keep`` stay; the others fill the slots
    given up below it.  Codes, params, weights and positions (int32, or None where a slot is its
    position) move together, in place or into ``out`` = (codes, params, weights, positions) of another
    cache.  ``seen``: int or int32 [B], by default ``length``.  Returns slots [B, NH, keep] int32: the
    row each slot holds afterwards, -1 where there is none."""
    B, NH, cap, D, si, sb, sh = _kv4_view(codes, params)
    dev = codes.device
    length, keep, recent = _int32("length", length), _int32("keep", keep), _int32("recent", recent)
    wp, wsb, wsh = _kv4_marks("weights", weights, torch.float32, B, NH, length, dev)
    if wp is None:
        raise ValueError("kv4_evict: weights are required")
    pp, psb, psh = _kv4_marks("positions", positions, torch.int32, B, NH, length, dev)
    if pp is not None and (psb, psh) != (wsb, wsh):
        raise ValueError("kv4_evict: weights and positions must have the same strides")
    dst = [None, None, None, None, 0, 0, 0, 0, 0, 0]
    if out is not None:
        oB, oNH, ocap, oD, osi, osb, osh = _kv4_view(out[0], out[1])
        if (oB, oNH, oD) != (B, NH, D) or out[0].device != dev:
            raise ValueError("kv4_evict: the destination's batch, heads or head_dim differ")
        ow, owsb, owsh = _kv4_marks("out weights", out[2], torch.float32, B, NH, keep, dev)
        op, opsb, opsh = _kv4_marks("out positions", out[3], torch.int32, B, NH, keep, dev)
        if op is not None and (opsb, opsh) != (owsb, owsh):
            raise ValueError("kv4_evict: the destination's weights and positions must have the same strides")
        dst = [out[0].data_ptr(), out[1].data_ptr(), ow, op, osi, osb, osh, ocap, owsb, owsh]
    if slots is None:
        slots = codes.new_empty((B, NH, max(keep, 0)), dtype=torch.int32)
    elif slots.shape != (B, NH, keep) or slots.dtype != torch.int32 or not slots.is_contiguous() or slots.device != dev:
        raise ValueError(f"slots: expected contiguous int32 [{B}, {NH}, {keep}] on {dev}")
    lengths_p = _row_counts("lengths", lengths, B, dev)
    if seen is None:
        seen = length if lengths is None else lengths
    seen_p, seen0 = _per_sequence("seen", seen, B, dev)
    if B == 0:
        return slots
    workspace, ws, ws_bytes = _scratch(workspace, _workspace_bytes("attn_kv4_evict_workspace_size", 0, B, NH, length, keep), codes)
    before = _other_device(dev)
    try:
        rc = lib.attn_kv4_evict(codes.data_ptr(), params.data_ptr(), wp, pp, si, sb, sh, cap, wsb, wsh, *dst,
                                B, NH, length, D, keep, recent, lengths_p, seen_p, seen0, slots.data_ptr(), ws, ws_bytes, _raw_stream(dev.index))
    finally:
        if before is not None:
            torch.cuda.set_device(before)
    if rc:
        raise AttnError("attn_kv4_evict", rc, last_error())
    return slots


def gemm(A: int, lda: int, a_trans: bool, B: int, ldb: int, b_trans: bool, ab_dtype: torch.dtype,
         C: int, ldc: int, c_dtype: torch.dtype, M: int, N: int, K: int, bias: int | None = None,
         accumulate: bool = False, max_ctas: int = 0):
    """C[M,N] (=|+=) op(A) op(B) (+bias) on raw device addresses (see include/attn_b200.h); on at
    most ``max_ctas`` SMs when it is positive (attn_gemm_ex)."""
    if max_ctas:
        call("attn_gemm_ex", A, lda, int(a_trans), B, ldb, int(b_trans), dtype_code(ab_dtype), C, ldc,
             dtype_code(c_dtype), bias, M, N, K, int(accumulate), int(max_ctas), _stream())
        return
    call("attn_gemm", A, lda, int(a_trans), B, ldb, int(b_trans), dtype_code(ab_dtype), C, ldc,
         dtype_code(c_dtype), bias, M, N, K, int(accumulate), _stream())


def gemm_act(A: int, lda: int, a_trans: bool, B: int, ldb: int, b_trans: bool, ab_dtype: torch.dtype,
             C: int, ldc: int, c_dtype: torch.dtype, M: int, N: int, K: int, act: int, aux: int | None = None,
             ldaux: int = 0, aux_dtype: torch.dtype = torch.float32, bias: int | None = None):
    """GEMM with the feed-forward activation in its epilogue (attn_gemm_act): ATTN_ACT_GELU writes
    gelu(op(A) op(B) + bias) to C and the pre-activation to aux; ATTN_ACT_GELU_BWD writes
    op(A) op(B) * gelu'(aux)."""
    call("attn_gemm_act", A, lda, int(a_trans), B, ldb, int(b_trans), dtype_code(ab_dtype), C, ldc,
         dtype_code(c_dtype), bias, M, N, K, int(act), aux, ldaux, dtype_code(aux_dtype), _stream())


def colsum(X: int, x_dtype: torch.dtype, ldx: int, M: int, N: int, out: torch.Tensor,
           accumulate: bool = False, workspace: torch.Tensor | None = None):
    need = lib.attn_colsum_workspace_size(M, N)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    call("attn_colsum", X, dtype_code(x_dtype), ldx, M, N, out.data_ptr(), int(accumulate),
         workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream())


def cast_colsum(x: torch.Tensor, colsum_out: torch.Tensor, accumulate: bool = False,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 copy of a float32 [M, N] matrix plus its column sums (into/onto colsum_out), one pass."""
    assert x.dtype == torch.float32 and x.is_contiguous() and x.dim() == 2
    M, N = x.shape
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=x.device)
    need = lib.attn_colsum_workspace_size(M, N)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    call("attn_cast_colsum_f32", x.data_ptr(), N, M, N, out.data_ptr(), N, colsum_out.data_ptr(),
         int(accumulate), workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream())
    return out


def cast_bf16(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    assert x.dtype == torch.float32 and x.is_contiguous()
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    call("attn_cast_f32_to_bf16", x.data_ptr(), out.data_ptr(), x.numel(), _stream())
    return out


def cast_rows_ones(x: torch.Tensor) -> torch.Tensor:
    """float32 [M, N] -> bf16 [M, L] with L = N + 1 rounded up to a multiple of 8 (16-byte rows):
    bf16(x), then a column of ones, then zeros.  Used as the QKV projection's input so the
    weight-gradient GEMM also yields the bias gradient."""
    assert x.dtype == torch.float32 and x.is_contiguous() and x.dim() == 2
    M, N = x.shape
    L = (N + 1 + 7) // 8 * 8
    out = torch.empty((M, L), dtype=torch.bfloat16, device=x.device)
    call("attn_cast_rows_ones_bf16", x.data_ptr(), N, M, N, out.data_ptr(), L, _stream())
    return out


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5,
              out_dtype: torch.dtype = torch.float32, ones_col: bool = False) -> torch.Tensor:
    """Row LayerNorm of float32 x [M, C] (layernorm_kernel, core/kernels.py:75-110) -> [M, C] in
    out_dtype, or, with ones_col (bf16), [M, L] = LN(x) | 1 | 0.. like cast_rows_ones."""
    assert x.dtype == torch.float32 and x.is_contiguous() and x.dim() == 2
    M, C = x.shape
    L = (C + 1 + 7) // 8 * 8 if ones_col else C
    out = torch.empty((M, L), dtype=out_dtype, device=x.device)
    call("attn_layernorm", x.data_ptr(), C, gamma.data_ptr(), beta.data_ptr(), M, C, float(eps), out.data_ptr(),
         L, dtype_code(out_dtype), int(ones_col), _stream())
    return out


def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, gamma: torch.Tensor, dx: torch.Tensor,
                       dgamma: torch.Tensor, dbeta: torch.Tensor, eps: float = 1e-5, accumulate_dx: bool = False,
                       accumulate_params: bool = False):
    """LayerNorm backward of layernorm_backward_kernel (core/kernels.py:361-416) on float32 [M, C]
    rows: dx (=|+=) dLN/dx, dgamma/dbeta (=|+=) the parameter gradients."""
    assert dy.dtype == x.dtype == dx.dtype == torch.float32 and dy.shape == x.shape == dx.shape
    M, C = x.shape
    call("attn_layernorm_bwd", dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), M, C, float(eps), dx.data_ptr(),
         int(accumulate_dx), dgamma.data_ptr(), dbeta.data_ptr(), int(accumulate_params), _stream())


def split_heads(qkv: int, q: int, k: int, v: int, B: int, T: int, NH: int, HD: int):
    """split_heads_kernel (core/mha_kernels.py:534-558) on float32 device buffers."""
    call("attn_split_heads", qkv, q, k, v, B, T, NH, HD, _stream())


def merge_heads(ctx_heads: int, ctx: int, B: int, T: int, NH: int, HD: int):
    """merge_heads_kernel (core/mha_kernels.py:567-584) on float32 device buffers."""
    call("attn_merge_heads", ctx_heads, ctx, B, T, NH, HD, _stream())


class _Kernel:
    """A named kernel handle shaped like the reference's PyCUDA functions (positional args)."""

    def __init__(self, name, fn):
        self.__name__ = name
        self._fn = fn

    def __call__(self, *args, block=None, grid=None, shared=None, stream=None):
        return self._fn(*[ptr(a) if not isinstance(a, (int, float)) else a for a in args])


class _SharedModule:
    """Stand-in for the compiled PyCUDA module of get_shared_mha_module (core/mha_ops.py:39-48):
    the layout adapters are exposed by the reference's kernel names."""

    def get_function(self, name):
        if name == "split_heads_kernel":
            return _Kernel(name, lambda qkv, q, k, v, B, T, NH, HD: split_heads(
                qkv, q, k, v, int(B), int(T), int(NH), int(HD)))
        if name == "merge_heads_kernel":
            return _Kernel(name, lambda ch, c, B, T, NH, HD: merge_heads(
                ch, c, int(B), int(T), int(NH), int(HD)))
        raise KeyError(f"{name}: the B200 library replaces this kernel; use MultiHeadAttention or "
                       "the attention_* wrappers")


_SHARED = _SharedModule()


def get_shared_mha_module():
    return _SHARED


class MHAController:
    """The reference's sandbox attention controller (core/mha_ops.py:55-138) on this library.

    ``forward(X[H, M, Din], W_qkv[Din, 3D])`` runs the fused-QKV causal attention pass on host
    float32 arrays and returns ``(out[H, M, D], probs[H, M, M])`` as the reference's does: the
    fused projection ``X W_qkv`` (matmul_qkv_fused, core/mha_kernels.py:689-720) is one float32
    GEMM; the reference's split into contiguous Q/K/V (split_qkv_kernel, :722-) is folded into the
    attention's strides (it reads Q, K and V straight out of the fused [H*M, 3D] buffer); the causal
    attention (fused_attention_forward_kernel) runs on the float32 kernels and writes the row
    log-sum-exp, from which ``probs`` is rebuilt on the device.  Inputs are copied to the device
    and the results back, as in the reference.  ``H, M, D`` fix the attention shape; ``module`` is
    accepted for signature compatibility.
    """

    def __init__(self, H: int, M: int, D: int, module=None):
        self.H, self.M, self.D = int(H), int(M), int(D)
        self.scale = 1.0 / math.sqrt(D)
        self.module = module if module is not None else get_shared_mha_module()

    def _fused(self, gX, gW, Din: int) -> torch.Tensor:
        H, M, D = self.H, self.M, self.D
        fused = torch.empty((H * M, 3 * D), dtype=torch.float32, device="cuda")
        gemm(gX.data_ptr(), Din, False, gW.data_ptr(), 3 * D, False, torch.float32, fused.data_ptr(), 3 * D,
             torch.float32, H * M, 3 * D, Din)
        return fused

    def matmul_qkv_fused(self, gpu_X, gpu_W, gpu_fused, Din: int, block=None, grid=None):
        """Fused[H, M, 3D] = X[H, M, Din] @ W_qkv[Din, 3D] on device buffers (the launch
        configuration arguments of the reference are accepted and unused)."""
        H, M, D = self.H, self.M, self.D
        gemm(ptr(gpu_X), Din, False, ptr(gpu_W), 3 * D, False, torch.float32, ptr(gpu_fused), 3 * D,
             torch.float32, H * M, 3 * D, int(Din))

    def forward(self, X, W_qkv):
        import numpy as np
        H, M, D = self.H, self.M, self.D
        X = np.ascontiguousarray(X, dtype=np.float32)
        W_qkv = np.ascontiguousarray(W_qkv, dtype=np.float32)
        if X.shape[:2] != (H, M) or W_qkv.shape != (X.shape[-1], 3 * D):
            raise ValueError(f"MHAController({H}, {M}, {D}): X {X.shape} / W_qkv {W_qkv.shape} do not match")
        Din = X.shape[-1]
        gX = torch.from_numpy(X).cuda().view(H * M, Din)
        gW = torch.from_numpy(W_qkv).cuda()
        fused = self._fused(gX, gW, Din)
        base, es = fused.data_ptr(), fused.element_size()
        # heads as batch entries of one head each: element (h, m, d) of Q/K/V at h*M*3D + m*3D + d
        qv, kv, vv = (HeadView(base + i * D * es, M * 3 * D, 3 * D, D) for i in range(3))
        out = torch.empty((H, M, D), dtype=torch.float32, device="cuda")
        lse = torch.empty((H, 1, M), dtype=torch.float32, device="cuda")
        attention_forward(qv, kv, vv, HeadView(out.data_ptr(), M * D, D, D), lse, H, 1, M, D, self.scale,
                          torch.float32)
        probs = attention_probs(qv, kv, lse, H, 1, M, D, self.scale, torch.float32)
        return out.cpu().numpy(), probs.view(H, M, M).cpu().numpy()
