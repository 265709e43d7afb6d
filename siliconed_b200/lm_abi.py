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

_lib = None
_TYPES = {torch.bfloat16: BF16, torch.float32: F32, torch.float8_e4m3fn: E4M3}


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
    _lib = lib
    return lib


def _check(status: int, what: str) -> None:
    if status != OK:
        raise LmError(f"{what}: status {status}", status)


def _need(what: str, ok: bool, message: str) -> None:
    if not ok:
        raise LmError(f"{what}: {message}")


def _take(what: str, name: str, t, device, dtypes, shape):
    """The tensor's address, after its device, dtype, shape (None: any size) and contiguity."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != len(shape) or \
            any(w is not None and w != s for w, s in zip(shape, t.shape)) or not t.is_contiguous() or t.device != device:
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)
        want = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        size = ", ".join("*" if w is None else str(w) for w in shape)
        raise LmError(f"{what}: {name} must be a contiguous {want} [{size}] tensor on {device}: got {got}")
    return t.data_ptr()


def _device(what: str, name: str, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise LmError(f"{what}: {name} must be a CUDA tensor")
    return t.device


def _call(fn: str, device, *args) -> None:
    """The call on `device` and its current stream."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        _check(getattr(load(), fn)(*args, stream), fn)
    else:
        with torch.cuda.device(device):
            _check(getattr(load(), fn)(*args, stream), fn)


_BF16, _F32, _I32, _E4M3, _FLOATS = (torch.bfloat16,), (torch.float32,), (torch.int32,), (torch.float8_e4m3fn,), \
    (torch.bfloat16, torch.float32)


def rms_norm_quantize(x, delta=None, weight=None, eps: float = 1e-6, x_out=None, codes=None, scales=None,
                      norm: bool = True):
    """z = x + delta; x_out = z (default: in place); RMSNorm(z) * weight as e4m3 codes with a scale per 128 values.

    x, delta: bf16 or fp32 [rows, d]; weight: fp32 [d].  Returns (x_out, codes float8_e4m3fn [rows, d], scales fp32
    [rows, ceil(d / 128)]).  ``norm=False`` quantizes z * weight itself.  Without ``delta`` x is not written.
    """
    what = "rms_norm_quantize"
    device = _device(what, "x", x)
    _need(what, x.dim() == 2, "x must be [rows, d]")
    rows, d = x.shape
    _need(what, d % 16 == 0 and 16 <= d <= 16384, f"d must be a multiple of 16 up to 16384: got {d}")
    blocks = -(-d // BLOCK)
    px = _take(what, "x", x, device, _FLOATS, (rows, d))
    pd = pw = None
    if delta is not None:
        pd = _take(what, "delta", delta, device, _FLOATS, (rows, d))
    if weight is not None:
        pw = _take(what, "weight", weight, device, _F32, (d,))
    if x_out is None:
        x_out = x
    _need(what, delta is not None or x_out is x, "x_out without delta must be x")
    po = _take(what, "x_out", x_out, device, (x.dtype,), (rows, d))
    if codes is None:
        codes = torch.empty(rows, d, dtype=torch.float8_e4m3fn, device=device)
    if scales is None:
        scales = torch.empty(rows, blocks, device=device)
    _call("sl_rms_norm_quantize", device, px, _TYPES[x.dtype], pd, BF16 if delta is None else _TYPES[delta.dtype], pw, eps,
          int(norm), rows, d, po, _take(what, "codes", codes, device, _E4M3, (rows, d)),
          _take(what, "scales", scales, device, _F32, (rows, blocks)))
    return x_out, codes, scales


def _cache(what, k_cache, v_cache, k_scale, v_scale, device, kv_heads, head_dim):
    """(type, pages, page size, the four addresses) of a paged cache."""
    _need(what, isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4,
          "k_cache must be [pages, kv_heads, page_size, head_dim]")
    pages, _, size, _ = k_cache.shape
    shape = (pages, kv_heads, size, head_dim)
    pk = _take(what, "k_cache", k_cache, device, _BF16 + _E4M3, shape)
    pv = _take(what, "v_cache", v_cache, device, (k_cache.dtype,), shape)
    if k_cache.dtype == torch.bfloat16:
        _need(what, k_scale is None and v_scale is None, "a bf16 cache has no scales")
        return BF16, pages, size, pk, pv, None, None
    return E4M3, pages, size, pk, pv, _take(what, "k_scale", k_scale, device, _F32, shape[:3]), \
        _take(what, "v_scale", v_scale, device, _F32, shape[:3])


def append_paged(qkv, heads: int, kv_heads: int, norm_q, norm_k, eps: float, freqs, pairs: str, seq, positions, table,
                 k_cache, v_cache, k_scale=None, v_scale=None, q=None):
    """QK-norm and rotation of new tokens; k and v into their page slots; returns q bf16 [tokens, heads, head_dim].

    qkv: bf16 [tokens, (heads + 2 kv_heads) * head_dim]; norm_q, norm_k: fp32 [head_dim] or None; freqs: fp32 [max_pos,
    head_dim / 2, 2] (cos, sin); pairs: "adjacent" or "halves"; seq: int32 [tokens] (None: token i is sequence i's);
    positions: int32 [tokens] (negative: padding); table: int32 [seqs, width]; caches [pages, kv_heads, page_size,
    head_dim], bf16, or float8_e4m3fn with fp32 scales [pages, kv_heads, page_size].
    """
    what = "append_paged"
    device = _device(what, "qkv", qkv)
    _need(what, heads >= 1 and kv_heads >= 1, "heads and kv_heads must be positive")
    _need(what, qkv.dim() == 2 and qkv.shape[1] % (heads + 2 * kv_heads) == 0, "qkv must be [tokens, (heads + 2 kv_heads) * head_dim]")
    tokens, dim = qkv.shape[0], qkv.shape[1] // (heads + 2 * kv_heads)
    _need(what, dim in (64, 128), f"head_dim must be 64 or 128: got {dim}")
    _need(what, pairs in PAIRS, f"pairs must be one of {sorted(PAIRS)}: got {pairs!r}")
    kind, pages, size, pk, pv, pks, pvs = _cache(what, k_cache, v_cache, k_scale, v_scale, device, kv_heads, dim)
    pf = _take(what, "freqs", freqs, device, _F32, (None, dim // 2, 2))
    pt = _take(what, "table", table, device, _I32, (None, None))
    seqs, width = table.shape
    _need(what, freqs.shape[0] > 0 and seqs > 0 and width > 0 and pages > 0 and size > 0, "an empty table, cache or freqs")
    _need(what, seq is not None or tokens <= seqs, f"{tokens} tokens for {seqs} sequences")
    if q is None:
        q = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=device)
    _call("sl_append_paged", device, _take(what, "qkv", qkv, device, _BF16, (tokens, None)), tokens, heads, kv_heads, dim,
          None if norm_q is None else _take(what, "norm_q", norm_q, device, _F32, (dim,)),
          None if norm_k is None else _take(what, "norm_k", norm_k, device, _F32, (dim,)), eps, pf, freqs.shape[0],
          PAIRS[pairs], None if seq is None else _take(what, "seq", seq, device, _I32, (tokens,)),
          _take(what, "positions", positions, device, _I32, (tokens,)), pt, seqs, width, pages, size, kind, pk, pv, pks, pvs,
          _take(what, "q", q, device, _BF16, (tokens, heads, dim)))
    return q


_workspaces: dict = {}


def attention_workspace(heads: int, kv_heads: int, head_dim: int, device=None):
    """A zeroed workspace for ``paged_attention``: one per stream whose calls may run at the same time."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    need = _SZ()
    with torch.cuda.device(device):
        _check(load().sl_paged_attention_workspace(heads, kv_heads, head_dim, ctypes.byref(need)),
               "sl_paged_attention_workspace")
        return torch.zeros(need.value, dtype=torch.uint8, device=device)


def _stream_workspace(heads, kv_heads, dim, device):
    """The current stream's workspace.  A call under graph capture gets one of its own, zeroed inside the graph: memory
    that only a replay writes must not be handed to later calls."""
    if torch.cuda.is_current_stream_capturing():
        return attention_workspace(heads, kv_heads, dim, device)
    key = (device.index, torch.cuda.current_stream(device).cuda_stream, heads // kv_heads > 8, dim)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = attention_workspace(heads, kv_heads, dim, device)
    return ws


def paged_attention(q, k_cache, v_cache, k_scale, v_scale, table, lengths, scale: float, out=None, lse=None, workspace=None):
    """softmax(scale q k^T) v of one new token per sequence over its first ``lengths`` cached tokens.

    q: bf16 [batch, heads, head_dim]; caches and scales as ``append_paged`` fills them; table: int32 [batch, width];
    lengths: int32 [batch], the new token counted.  Returns ``out`` (bf16, like q); ``lse`` (fp32 [batch, heads], when
    given) is filled with log sum exp.  A sequence of length 0 gives zeros and -inf.
    """
    what = "paged_attention"
    device = _device(what, "q", q)
    _need(what, q.dim() == 3, "q must be [batch, heads, head_dim]")
    batch, heads, dim = q.shape
    _need(what, dim in (64, 128), f"head_dim must be 64 or 128: got {dim}")
    _need(what, isinstance(k_cache, torch.Tensor) and k_cache.dim() == 4, "k_cache must be [pages, kv_heads, page_size, head_dim]")
    kv_heads = k_cache.shape[1]
    _need(what, kv_heads > 0 and heads > 0 and heads % kv_heads == 0, f"{kv_heads} key-value heads for {heads} query heads")
    kind, pages, size, pk, pv, pks, pvs = _cache(what, k_cache, v_cache, k_scale, v_scale, device, kv_heads, dim)
    pt = _take(what, "table", table, device, _I32, (batch, None))
    width = table.shape[1]
    _need(what, width > 0 and pages > 0 and size > 0, "an empty table or cache")
    if out is None:
        out = torch.empty_like(q)
    if workspace is None:
        workspace = _stream_workspace(heads, kv_heads, dim, device)
    _call("sl_paged_attention", device, _take(what, "q", q, device, _BF16, (batch, heads, dim)), pk, pv, pks, pvs, kind, pt,
          _take(what, "lengths", lengths, device, _I32, (batch,)), batch, heads, kv_heads, dim, width, pages, size, scale,
          _take(what, "out", out, device, _BF16, (batch, heads, dim)),
          None if lse is None else _take(what, "lse", lse, device, _F32, (batch, heads)),
          _take(what, "workspace", workspace, device, (torch.uint8,), (None,)), workspace.numel())
    return out


def linear_block_fp8(codes, scales, weight, weight_scales, bias=None, out=None):
    """out[m, n] = (codes * scales) . (weight * weight_scales)^T + bias, scales per 128 and per 128 x 128 values.

    codes: float8_e4m3fn [m, k] and scales fp32 [m, ceil(k / 128)] (``rms_norm_quantize``); weight: float8_e4m3fn [n, k]
    as published, weight_scales fp32 [ceil(n / 128), ceil(k / 128)]; bias: bf16 [n]; out: bf16 (default) or fp32 [m, n].
    """
    what = "linear_block_fp8"
    device = _device(what, "codes", codes)
    _need(what, codes.dim() == 2 and isinstance(weight, torch.Tensor) and weight.dim() == 2, "codes must be [m, k], weight [n, k]")
    (m, k), n = codes.shape, weight.shape[0]
    _need(what, k >= 16 and k % 16 == 0 and n > 0, f"k must be a multiple of 16 and n positive: got k {k}, n {n}")
    kb, nb = -(-k // BLOCK), -(-n // BLOCK)
    if out is None:
        out = torch.empty(m, n, dtype=torch.bfloat16, device=device)
    _call("sl_linear_block_fp8", device, _take(what, "codes", codes, device, _E4M3, (m, k)),
          _take(what, "scales", scales, device, _F32, (m, kb)), _take(what, "weight", weight, device, _E4M3, (n, k)),
          _take(what, "weight_scales", weight_scales, device, _F32, (nb, kb)),
          None if bias is None else _take(what, "bias", bias, device, _BF16, (n,)), m, n, k,
          _take(what, "out", out, device, _FLOATS, (m, n)), _TYPES[out.dtype])
    return out


def errors(device=None) -> tuple[int, int]:
    """(status, site) of the library's device error word since the last call, after a wait for the device: (OK, 0), or
    OUT_OF_RANGE / TIMEOUT and its place."""
    site = _I(0)
    with torch.cuda.device(torch.cuda.current_device() if device is None else device):
        return load().sl_errors(ctypes.byref(site)), site.value
