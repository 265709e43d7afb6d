"""ctypes bindings of libsiliconed_lm.so (include/siliconed_lm.h), and tensor-level wrappers.

The library carries a decoder layer's operators beside its 8-bit linears: the residual addition, RMS norm and
quantization to e4m3; the product of such codes with a block-scaled e4m3 weight; the append to a paged key-value cache;
and the attention of one new token per sequence over that cache.  The wrappers take contiguous CUDA tensors of one
device and run on its current stream; what does not fit raises ``LmError``.
"""
from __future__ import annotations

import ctypes
import os
import re
import struct

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsiliconed_lm.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "siliconed_lm.h")

OK, INVALID_ARG, CUDA_ERROR, TIMEOUT, OUT_OF_RANGE = 0, 1, 4, 5, 10
BF16, F32, E4M3 = 0, 1, 2
PAIRS = {"adjacent": 0, "halves": 1}
BLOCK = 128

_P, _I, _I64, _F, _SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t

SIGNATURES = {
    "sl_rms_norm_quantize": (_I, [_P, _I, _P, _I, _P, _F, _I, _I64, _I, _P, _P, _P, _P]),
    "sl_append_paged": (_I, [_P, _I64, _I, _I, _I, _P, _P, _F, _P, _I, _I, _P, _P, _P, _I, _I, _I64, _I, _I, _P, _P, _P, _P,
                             _P, _P]),
    "sl_paged_attention_workspace": (_I, [_I, _I, _I, ctypes.POINTER(_SZ)]),
    "sl_paged_attention": (_I, [_P, _P, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I64, _I, _F, _P, _P, _P, _SZ, _P]),
    "sl_linear_block_fp8": (_I, [_P, _P, _P, _P, _P, _I64, _I64, _I64, _P, _I, _P]),
    "sl_errors": (_I, [ctypes.POINTER(_I)]),
}
# The operators' calls with their arguments packed into a C struct: every argument of a ctypes call costs.
_CODES = {_P: "P", _I: "i", _I64: "q", _F: "f", _SZ: "N"}
_PACKED = {name: struct.Struct("@" + "".join(_CODES[t] for t in SIGNATURES[name][1]))
           for name in ("sl_rms_norm_quantize", "sl_append_paged", "sl_paged_attention", "sl_linear_block_fp8")}
SIGNATURES.update({name + "_with": (_I, [ctypes.c_char_p]) for name in _PACKED})

_lib = None
_calls: dict = {}


class LmError(RuntimeError):
    """A refused argument, or a status of the library that is not SL_OK."""

    def __init__(self, message: str, status: int = INVALID_ARG):
        self.status = status
        super().__init__(message)


def header_functions() -> set[str]:
    text = open(HEADER).read()
    return set(re.findall(r"^SL_API\s+\w+\s+(sl_\w+)\s*\(", text, flags=re.M))


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        from . import build as _build
        _build.build()
    lib = ctypes.CDLL(path)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _calls.update({name: (getattr(lib, name + "_with"), form.pack) for name, form in _PACKED.items()})
    _lib = lib
    return lib


def _check(status: int, what: str) -> None:
    if status != OK:
        raise LmError(f"{what}: status {status}", status)


def _refuse(what: str, name: str, t, dtypes, shape, index: int):
    got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)
    want = " or ".join(str(d).replace("torch.", "") for d in dtypes)
    size = ", ".join("*" if w is None else str(w) for w in shape)
    raise LmError(f"{what}: {name} must be a contiguous {want} [{size}] tensor on cuda:{index}: got {got}")


def _take(what: str, name: str, t, dtype, shape, index: int) -> int:
    """The tensor's address, after its dtype, shape, contiguity and device.  (Called for every operand of every call: the
    message is made only on the way out.)"""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or t.get_device() != index or \
            not t.is_contiguous():
        _refuse(what, name, t, (dtype,), shape, index)
    return t.data_ptr()


def _index(what: str, name: str, t, dims: int) -> int:
    """The device index of the operand that names the call's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != dims:
        raise LmError(f"{what}: {name} must be a CUDA tensor of {dims} dimensions")
    return t.get_device()


def _call(fn: str, index: int, *args) -> None:
    """The call on device `index` and its current stream; a null pointer is 0."""
    if _lib is None:
        load()
    call, pack = _calls[fn]
    try:
        if index == torch._C._cuda_getDevice():
            status = call(pack(*args, torch._C._cuda_getCurrentRawStream(index)))
        else:
            with torch.cuda.device(index):
                status = call(pack(*args, torch._C._cuda_getCurrentRawStream(index)))
    except (struct.error, OverflowError) as e:
        raise LmError(f"{fn}: {e}") from None
    if status != OK:
        raise LmError(f"{fn}: status {status}", status)


_BF16, _F32, _I32, _E4M3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn


def rms_norm_quantize(x, delta=None, weight=None, eps: float = 1e-6, x_out=None, codes=None, scales=None,
                      norm: bool = True):
    """z = x + delta; x_out = z (default: in place); RMSNorm(z) * weight as e4m3 codes with a scale per 128 values.

    x, delta: bf16 or fp32 [rows, d]; weight: fp32 [d].  Returns (x_out, codes float8_e4m3fn [rows, d], scales fp32
    [rows, ceil(d / 128)]).  ``norm=False`` quantizes z * weight itself.  Without ``delta`` x is not written.
    """
    what = "rms_norm_quantize"
    index = _index(what, "x", x, 2)
    shape = x.shape
    rows, d = shape
    if d % 16 != 0 or d < 16 or d > 16384:
        raise LmError(f"{what}: d must be a multiple of 16 up to 16384: got {d}")
    blocks = (rows, (d + BLOCK - 1) // BLOCK)
    if x.dtype is not _F32 and x.dtype is not _BF16:
        _refuse(what, "x", x, (_BF16, _F32), shape, index)
    px = po = _take(what, "x", x, x.dtype, shape, index)
    pd = pw = 0
    kind = BF16
    if delta is not None:
        kind = F32 if getattr(delta, "dtype", None) is _F32 else BF16
        pd = _take(what, "delta", delta, _F32 if kind == F32 else _BF16, shape, index)
        if x_out is not None:
            po = _take(what, "x_out", x_out, x.dtype, shape, index)
    elif x_out is not None and x_out is not x:
        raise LmError(f"{what}: x_out without delta must be x")
    if weight is not None:
        pw = _take(what, "weight", weight, _F32, (d,), index)
    if codes is None:
        codes = torch.empty(rows, d, dtype=_E4M3, device=x.device)
    if scales is None:
        scales = torch.empty(blocks, device=x.device)
    _call("sl_rms_norm_quantize", index, px, F32 if x.dtype is _F32 else BF16, pd, kind, pw, eps, int(norm), rows, d, po,
          _take(what, "codes", codes, _E4M3, shape, index), _take(what, "scales", scales, _F32, blocks, index))
    return x if x_out is None else x_out, codes, scales


def _cache(what, k_cache, v_cache, k_scale, v_scale, index, kv_heads, head_dim):
    """(type, pages, page size, the four addresses) of a paged cache."""
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 4:
        raise LmError(f"{what}: k_cache must be [pages, kv_heads, page_size, head_dim]")
    pages, _, size, _ = k_cache.shape
    shape = (pages, kv_heads, size, head_dim)
    if pages == 0 or size == 0:
        raise LmError(f"{what}: an empty cache")
    if k_cache.dtype is _BF16:
        if k_scale is not None or v_scale is not None:
            raise LmError(f"{what}: a bf16 cache has no scales")
        return BF16, pages, size, _take(what, "k_cache", k_cache, _BF16, shape, index), \
            _take(what, "v_cache", v_cache, _BF16, shape, index), 0, 0
    return E4M3, pages, size, _take(what, "k_cache", k_cache, _E4M3, shape, index), \
        _take(what, "v_cache", v_cache, _E4M3, shape, index), _take(what, "k_scale", k_scale, _F32, shape[:3], index), \
        _take(what, "v_scale", v_scale, _F32, shape[:3], index)


def append_paged(qkv, heads: int, kv_heads: int, norm_q, norm_k, eps: float, freqs, pairs: str, seq, positions, table,
                 k_cache, v_cache, k_scale=None, v_scale=None, q=None):
    """QK-norm and rotation of new tokens; k and v into their page slots; returns q bf16 [tokens, heads, head_dim].

    qkv: bf16 [tokens, (heads + 2 kv_heads) * head_dim]; norm_q, norm_k: fp32 [head_dim] or None; freqs: fp32 [max_pos,
    head_dim / 2, 2] (cos, sin); pairs: "adjacent" or "halves"; seq: int32 [tokens] (None: token i is sequence i's);
    positions: int32 [tokens] (negative: padding); table: int32 [seqs, width]; caches [pages, kv_heads, page_size,
    head_dim], bf16, or float8_e4m3fn with fp32 scales [pages, kv_heads, page_size].
    """
    what = "append_paged"
    index = _index(what, "qkv", qkv, 2)
    if heads < 1 or kv_heads < 1 or qkv.shape[1] % (heads + 2 * kv_heads) != 0:
        raise LmError(f"{what}: qkv must be [tokens, (heads + 2 kv_heads) * head_dim]")
    tokens, dim = qkv.shape[0], qkv.shape[1] // (heads + 2 * kv_heads)
    if dim != 128 and dim != 64:
        raise LmError(f"{what}: head_dim must be 64 or 128: got {dim}")
    if pairs not in PAIRS:
        raise LmError(f"{what}: pairs must be one of {sorted(PAIRS)}: got {pairs!r}")
    kind, pages, size, pk, pv, pks, pvs = _cache(what, k_cache, v_cache, k_scale, v_scale, index, kv_heads, dim)
    if not isinstance(freqs, torch.Tensor) or freqs.dim() != 3 or not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise LmError(f"{what}: freqs must be [max_pos, head_dim / 2, 2], table [seqs, width]")
    max_pos, (seqs, width) = freqs.shape[0], table.shape
    if max_pos == 0 or width == 0 or (seqs == 0 and tokens != 0):
        raise LmError(f"{what}: an empty table or freqs")
    if seq is None and tokens > seqs:
        raise LmError(f"{what}: {tokens} tokens for {seqs} sequences")
    if q is None:
        q = torch.empty(tokens, heads, dim, dtype=_BF16, device=qkv.device)
    _call("sl_append_paged", index, _take(what, "qkv", qkv, _BF16, qkv.shape, index), tokens, heads, kv_heads, dim,
          0 if norm_q is None else _take(what, "norm_q", norm_q, _F32, (dim,), index),
          0 if norm_k is None else _take(what, "norm_k", norm_k, _F32, (dim,), index), eps,
          _take(what, "freqs", freqs, _F32, (max_pos, dim // 2, 2), index), max_pos, PAIRS[pairs],
          0 if seq is None else _take(what, "seq", seq, _I32, (tokens,), index),
          _take(what, "positions", positions, _I32, (tokens,), index), _take(what, "table", table, _I32, (seqs, width), index),
          seqs, width, pages, size, kind, pk, pv, pks, pvs, _take(what, "q", q, _BF16, (tokens, heads, dim), index))
    return q


_workspaces: dict = {}
_MOST_WORKSPACES = 16  # 2 to 10 MB each


def attention_workspace(heads: int, kv_heads: int, head_dim: int, device=None):
    """A zeroed workspace for ``paged_attention``: one per stream whose calls may run at the same time."""
    device = torch.device("cuda", torch.cuda.current_device() if device is None else device) \
        if device is None or isinstance(device, int) else torch.device(device)
    need = _SZ()
    with torch.cuda.device(device):
        _check(load().sl_paged_attention_workspace(heads, kv_heads, head_dim, ctypes.byref(need)),
               "sl_paged_attention_workspace")
        return torch.zeros(need.value, dtype=torch.uint8, device=device)


def _stream_workspace(heads, kv_heads, dim, index):
    """The current stream's workspace, of which the latest few are kept: a program may make streams as it goes.  (One that is
    dropped goes back to the allocator for its own stream, behind the calls that use it.)  A call under graph capture gets one
    of its own, zeroed inside the graph: memory that only a replay writes must not be handed to later calls."""
    if torch.cuda.is_current_stream_capturing():
        return attention_workspace(heads, kv_heads, dim, index)
    key = (index, torch._C._cuda_getCurrentRawStream(index), heads > 8 * kv_heads, dim)
    ws = _workspaces.get(key)
    if ws is None:
        while len(_workspaces) >= _MOST_WORKSPACES:
            _workspaces.pop(next(iter(_workspaces)), None)
        ws = _workspaces[key] = attention_workspace(heads, kv_heads, dim, index)
    return ws


def paged_attention(q, k_cache, v_cache, k_scale, v_scale, table, lengths, scale: float, out=None, lse=None, workspace=None):
    """softmax(scale q k^T) v of one new token per sequence over its first ``lengths`` cached tokens.

    q: bf16 [batch, heads, head_dim]; caches and scales as ``append_paged`` fills them; table: int32 [batch, width];
    lengths: int32 [batch], the new token counted.  Returns ``out`` (bf16, like q); ``lse`` (fp32 [batch, heads], when
    given) is filled with log sum exp.  A sequence of length 0 gives zeros and -inf.
    """
    what = "paged_attention"
    index = _index(what, "q", q, 3)
    shape = q.shape
    batch, heads, dim = shape
    if dim != 128 and dim != 64:
        raise LmError(f"{what}: head_dim must be 64 or 128: got {dim}")
    kv_heads = k_cache.shape[1] if isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4 else 0
    if kv_heads < 1 or heads < 1 or heads % kv_heads != 0:
        raise LmError(f"{what}: {kv_heads} key-value heads for {heads} query heads")
    kind, pages, size, pk, pv, pks, pvs = _cache(what, k_cache, v_cache, k_scale, v_scale, index, kv_heads, dim)
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.shape[1] == 0:
        raise LmError(f"{what}: table must be [batch, width]")
    width = table.shape[1]
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = _stream_workspace(heads, kv_heads, dim, index)
    space = workspace.numel() if isinstance(workspace, torch.Tensor) else 0
    _call("sl_paged_attention", index, _take(what, "q", q, _BF16, shape, index), pk, pv, pks, pvs, kind,
          _take(what, "table", table, _I32, (batch, width), index), _take(what, "lengths", lengths, _I32, (batch,), index),
          batch, heads, kv_heads, dim, width, pages, size, scale, _take(what, "out", out, _BF16, shape, index),
          0 if lse is None else _take(what, "lse", lse, _F32, (batch, heads), index),
          _take(what, "workspace", workspace, torch.uint8, (space,), index), space)
    return out


def linear_block_fp8(codes, scales, weight, weight_scales, bias=None, out=None):
    """out[m, n] = (codes * scales) . (weight * weight_scales)^T + bias, scales per 128 and per 128 x 128 values.

    codes: float8_e4m3fn [m, k] and scales fp32 [m, ceil(k / 128)] (``rms_norm_quantize``); weight: float8_e4m3fn [n, k]
    as published, weight_scales fp32 [ceil(n / 128), ceil(k / 128)]; bias: bf16 [n]; out: bf16 (default) or fp32 [m, n].
    """
    what = "linear_block_fp8"
    index = _index(what, "codes", codes, 2)
    m, k = codes.shape
    n = weight.shape[0] if isinstance(weight, torch.Tensor) and weight.dim() == 2 else 0
    if k < 16 or k % 16 != 0 or n < 1:
        raise LmError(f"{what}: codes must be [m, k], weight [n, k], k a multiple of 16: got k {k}, n {n}")
    kb, nb = (k + BLOCK - 1) // BLOCK, (n + BLOCK - 1) // BLOCK
    if out is None:
        out = torch.empty(m, n, dtype=_BF16, device=codes.device)
    kind = F32 if getattr(out, "dtype", None) is _F32 else BF16
    _call("sl_linear_block_fp8", index, _take(what, "codes", codes, _E4M3, (m, k), index),
          _take(what, "scales", scales, _F32, (m, kb), index), _take(what, "weight", weight, _E4M3, (n, k), index),
          _take(what, "weight_scales", weight_scales, _F32, (nb, kb), index),
          0 if bias is None else _take(what, "bias", bias, _BF16, (n,), index), m, n, k,
          _take(what, "out", out, _F32 if kind == F32 else _BF16, (m, n), index), kind)
    return out


def errors(device=None) -> tuple[int, int]:
    """(status, site) of the library's device error word since the last call, after a wait for the device: (OK, 0), or
    OUT_OF_RANGE / TIMEOUT and its place."""
    site = _I(0)
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        return load().sl_errors(ctypes.byref(site)), site.value
