"""Host-side operators on torch tensors: thin, allocation-explicit wrappers over the C ABI.

These mirror how the reference reaches an external kernel: destination-passing packed
functions on DLPack tensors (``R.call_tir("b200.q4f16_matmul", (x, wq, scales), out_sinfo)``;
reference: python/tvm/relax/op/base.py:47-91, src/relax/transform/call_tir_rewrite.cc:55-116).
torch is used only for device memory and streams.
"""
from __future__ import annotations

import ctypes
import importlib.util
import typing

import torch

from . import _lib, build
from ._lib import B200Error, DLDataType, DLDevice, DLTensor  # noqa: F401


import contextlib


def _stream_ptr(device) -> int:
    if torch.device(device).type != "cuda":
        return 0
    return torch.cuda.current_stream(device).cuda_stream


def _on(device):
    """Makes `device` current for the call; a CPU tensor is passed through so that the library's
    own validation rejects it (there is no host implementation to fall back to)."""
    return torch.cuda.device(device) if torch.device(device).type == "cuda" else contextlib.nullcontext()


_DTYPES = {
    torch.float16: (2, 16),
    torch.float32: (2, 32),
    torch.uint32: (1, 32),
    torch.int32: (0, 32),
    torch.uint8: (1, 8),
}


class _DLView:
    """Keeps the ctypes arrays of a DLTensor view alive."""

    def __init__(self, t: torch.Tensor):
        code, bits = _DTYPES[t.dtype]
        self.shape = (ctypes.c_int64 * t.dim())(*t.shape)
        self.strides = (ctypes.c_int64 * t.dim())(*t.stride())
        if t.is_cuda:
            dev = DLDevice(2, t.device.index if t.device.index is not None else torch.cuda.current_device())
        else:
            dev = DLDevice(1, 0)
        self.tensor = DLTensor(
            ctypes.c_void_p(t.data_ptr()), dev, t.dim(), DLDataType(code, bits, 1),
            ctypes.cast(self.shape, ctypes.POINTER(ctypes.c_int64)),
            ctypes.cast(self.strides, ctypes.POINTER(ctypes.c_int64)), 0,
        )
        self.keep = t

    def ptr(self):
        return ctypes.byref(self.tensor)


def to_dltensor(t: torch.Tensor) -> _DLView:
    return _DLView(t)


LAYOUTS = {"reference": _lib.LAYOUT_REFERENCE, "paired": _lib.LAYOUT_PAIRED}


def _layout_code(layout) -> int:
    if isinstance(layout, str):
        if layout not in LAYOUTS:
            raise ValueError(f"unknown weight layout {layout!r}; one of {sorted(LAYOUTS)}")
        return LAYOUTS[layout]
    return int(layout)


class _option_scope:
    """Sets a process-wide option of the library for the duration of a block."""

    def __init__(self, name: str, value: int):
        self.name, self.value = name, value

    def __enter__(self):
        L = _lib.lib()
        self.saved = L.b200_get_option(self.name.encode())
        _lib.check(L.b200_set_option(self.name.encode(), self.value))

    def __exit__(self, *exc):
        _lib.check(_lib.lib().b200_set_option(self.name.encode(), self.saved))


_F16, _U32 = torch.float16, torch.uint32


def _plain(device, *tensors) -> bool:
    """True when the tensors are contiguous 2-D tensors on the current CUDA device, so that their pointers and shapes
    say all that a DLPack view would."""
    for t in tensors:
        if t.device != device or t.dim() != 2 or not t.is_contiguous():
            return False
    return device.type == "cuda" and torch._C._cuda_getDevice() == device.index


def _matmul_by_pointer(L, x, wq, scales, out, layout) -> bool:
    """The call through the raw-pointer entry point: what the DLPack entry point checks is checked here (a handful of
    attribute reads) instead of being marshalled into four ctypes structures, which took 25 of a call's 30 us.  False:
    nothing has been launched, the DLPack entry point takes the call or names the error."""
    if x.dtype is not _F16 or wq.dtype is not _U32 or scales.dtype is not _F16 or out.dtype is not _F16:
        return False
    device = x.device
    if not _plain(device, x, wq, scales, out):
        return False
    m, k = x.shape
    n = wq.shape[0]
    if k % 32 or wq.shape[1] * 8 != k or scales.shape != (n, k // 32) or out.shape != (m, n):
        return False
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    L.b200_set_stream(stream)
    if layout is None:
        return L.b200_q4f16_matmul(x.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(), m, n, k, stream) == 0
    return L.b200_q4f16_matmul_layout(x.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(), m, n, k,
                                      _layout_code(layout), stream) == 0


def _dequantize_by_pointer(L, wq, scales, out) -> bool:
    """As :func:`_matmul_by_pointer`, for the decode stage alone."""
    if wq.dtype is not _U32 or scales.dtype is not _F16 or out.dtype is not _F16:
        return False
    device = wq.device
    if not _plain(device, wq, scales, out):
        return False
    n, k = wq.shape[0], wq.shape[1] * 8
    if k % 32 or scales.shape != (n, k // 32) or out.shape != (n, k):
        return False
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    L.b200_set_stream(stream)
    return L.b200_q4f16_dequantize(wq.data_ptr(), scales.data_ptr(), out.data_ptr(), n, k, stream) == 0


_native = None      # the extension module, bound to the loaded library; False: not built for this torch (the checks run in Python then)


def _torch_call():
    global _native
    if _native is None:
        path = build.torch_call_path(torch.__version__)
        try:
            spec = importlib.util.spec_from_file_location(__package__ + "._torch_call", path)
            module = importlib.util.module_from_spec(spec)
        except ImportError:                 # (no such file, or one that does not load)
            _native = False
        else:
            L = _lib.lib()
            module.bind(*(ctypes.cast(fn, ctypes.c_void_p).value
                          for fn in (L.b200_set_stream, L.b200_q4f16_matmul, L.b200_q4f16_matmul_layout, L.b200_q4f16_dequantize,
                                     L.b200_paged_rope_append, L.b200_paged_attention, L.b200_token_logprobs)))
            _native = module
    return _native


def q4f16_matmul(x: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None,
                 family: str = "auto", layout=None) -> torch.Tensor:
    """y[M,N] fp16 = x[M,K] . decode(wq[N,K/8], scales[N,K/32])^T.  Plain contiguous tensors on the current device go
    straight to the raw-pointer entry point (through the extension, or with the same checks in Python); everything else goes
    through the DLPack entry point, which validates it and names the error.  ``family`` = "auto" | "gemv" | "gemm" picks the raw
    entry point of one kernel family instead.  ``layout`` ("reference" | "paired") names the nibble order
    of ``wq`` for this call; None takes the library's option "weights.layout"."""
    if out is None:
        out = torch.empty((x.shape[0], wq.shape[0]), dtype=torch.float16, device=x.device)
    if family == "auto":
        native = _native or _torch_call()
        if native and native.matmul(x, wq, scales, out, -1 if layout is None else _layout_code(layout)):
            return out
    L = _lib.lib()
    if family == "auto":
        if _matmul_by_pointer(L, x, wq, scales, out, layout):
            return out
        with _on(x.device):
            L.b200_set_stream(_stream_ptr(x.device))
            vx, vw, vs, vy = (_DLView(t) for t in (x, wq, scales, out))
            if layout is None:
                _lib.check(L.b200_q4f16_matmul_dl(vx.ptr(), vw.ptr(), vs.ptr(), vy.ptr()))
            else:
                code = _lib.family_with_layout(_lib.FAMILY_AUTO, _layout_code(layout))
                _lib.check(L.b200_q4f16_matmul_dl_family(vx.ptr(), vw.ptr(), vs.ptr(), vy.ptr(), code))
        return out
    fn = {"gemv": L.b200_q4f16_gemv, "gemm": L.b200_q4f16_gemm, "gemm_ws": L.b200_q4f16_gemm_ws,
          "matmul": L.b200_q4f16_matmul}[family]
    M, K = x.shape
    N = wq.shape[0]
    with _on(x.device):
        if layout is None:
            _lib.check(fn(x.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(), M, N, K, _stream_ptr(x.device)))
        else:
            with _option_scope("weights.layout", _layout_code(layout)):
                _lib.check(fn(x.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(), M, N, K, _stream_ptr(x.device)))
    return out


def q4f16_repack(wq: torch.Tensor, layout="paired", out: torch.Tensor | None = None) -> torch.Tensor:
    """The packed words of ``wq`` (reference nibble order) in ``layout``; ``out`` may be ``wq`` itself."""
    return _repack(wq, layout, out, to_layout=True)


def q4f16_unpack(packed: torch.Tensor, layout="paired", out: torch.Tensor | None = None) -> torch.Tensor:
    """Back to the reference's nibble order: the exact inverse of :func:`q4f16_repack`."""
    return _repack(packed, layout, out, to_layout=False)


def _repack(src: torch.Tensor, layout, out, to_layout: bool) -> torch.Tensor:
    if src.dtype not in (torch.int32, torch.uint32) or src.dim() != 2 or not src.is_contiguous():
        raise ValueError("packed weights are a contiguous 2-D 32-bit integer tensor [N, K/8]")
    if out is None:
        out = torch.empty_like(src)
    if out.shape != src.shape or out.dtype != src.dtype or out.device != src.device or not out.is_contiguous():
        raise ValueError("out must match the packed tensor")
    L = _lib.lib()
    fn = L.b200_q4f16_repack if to_layout else L.b200_q4f16_unpack
    N, K = src.shape[0], src.shape[1] * 8
    with _on(src.device):
        _lib.check(fn(src.data_ptr(), out.data_ptr(), N, K, _layout_code(layout), _stream_ptr(src.device)))
    return out


def q4f16_dequantize(wq: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None, layout=None) -> torch.Tensor:
    """w[N,K] fp16 = decode(wq, scales); bit-exact with the reference's decode stage."""
    if out is None:
        out = torch.empty((wq.shape[0], wq.shape[1] * 8), dtype=torch.float16, device=wq.device)
    if layout is None:
        native = _native or _torch_call()
        if native and native.dequantize(wq, scales, out):
            return out
    L = _lib.lib()
    if layout is not None:
        N, K = wq.shape[0], wq.shape[1] * 8
        with _on(wq.device):
            _lib.check(L.b200_q4f16_dequantize_layout(wq.data_ptr(), scales.data_ptr(), out.data_ptr(), N, K,
                                                      _layout_code(layout), _stream_ptr(wq.device)))
        return out
    if _dequantize_by_pointer(L, wq, scales, out):
        return out
    with _on(wq.device):
        L.b200_set_stream(_stream_ptr(wq.device))
        vw, vs, vo = (_DLView(t) for t in (wq, scales, out))
        _lib.check(L.b200_q4f16_dequantize_dl(vw.ptr(), vs.ptr(), vo.ptr()))
    return out


# ---------------------------------------------------------------------------------------------- paged key-value cache
_CACHE_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_LOGIT_TYPES = {**_CACHE_TYPES, torch.float32: _lib.F32}


def _same_device(device, **tensors):
    if device.type != "cuda":
        raise ValueError("the tensors must be on a CUDA device: there is no host implementation")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, other arguments on {device}")


def _index(name, t, shape):
    if t is None:
        return None
    if t.dtype is not torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _paged_cache(rows, k_pages, v_pages, page_table, lengths, starts, max_query) -> _lib.PagedCache:
    """The descriptor of a call over `rows` (whose first dimension is the tokens of the call), its tensors checked."""
    if k_pages.dtype not in _CACHE_TYPES or v_pages.dtype is not k_pages.dtype:
        raise ValueError(f"pages are fp16 or bf16, both alike: got {k_pages.dtype} and {v_pages.dtype}")
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise ValueError(f"pages are [pages, kv_heads, page_size, head_dim], both alike: got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    pages, kv_heads, page_size, head_dim = k_pages.shape
    whole = kv_heads * page_size * head_dim             # (the stride of a dimension of one entry says nothing)
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.stride()[2:] != (head_dim, 1) or (kv_heads > 1 and t.stride(1) != page_size * head_dim):
            raise ValueError(f"the heads of a page of {name} must be contiguous: strides {t.stride()}")
    if page_table.dtype is not torch.int32 or page_table.dim() != 2 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table is an int32 tensor [batch, pages of the longest sequence] with contiguous rows")
    batch, width = page_table.shape
    tokens = rows.shape[0]
    if starts is None:
        max_query = 1
        if tokens != batch:
            raise ValueError(f"{tokens} rows of {batch} sequences: without starts every sequence has one row")
    elif max_query is None:
        max_query = tokens
    stride = page_table.stride(0) if batch > 1 else width
    return _lib.PagedCache(_CACHE_TYPES[k_pages.dtype], kv_heads, head_dim, page_size, pages,
                           *(t.stride(0) if pages > 1 else whole for t in (k_pages, v_pages)), k_pages.data_ptr(), v_pages.data_ptr(), batch, width, int(max_query), stride, tokens, page_table.data_ptr(),
                           _index("lengths", lengths, (batch,)), _index("starts", starts, (batch + 1,)))


def paged_rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      page_table: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor | None = None, interleaved: bool = False,
                      positions: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q and k of qkv [tokens, (heads + 2 kv_heads) * head_dim] by their positions, stores k and v in the pages and returns
    q [tokens, heads, head_dim].

    ``lengths`` [batch] counts the tokens of every sequence with the new ones; rows ``starts[b] .. starts[b + 1] - 1`` are the newest of
    sequence b (None: one row each).  cos and sin, fp32 [positions, r / 2], turn the first r values of a head: pairs (i, i + r / 2), or
    (2 i, 2 i + 1) with ``interleaved``; ``positions`` (int32 [tokens]) names other rows of the tables than the tokens' places."""
    native = _native or _torch_call()
    if native:
        q = native.paged_rope_append(qkv, cos, sin, k_pages, v_pages, page_table, lengths, starts, interleaved, positions, out)
        if q is not None:
            return q
    cache = _paged_cache(qkv, k_pages, v_pages, page_table, lengths, starts, 1)
    kv, dim = cache.kv_heads, cache.head_dim
    if qkv.dtype is not k_pages.dtype or qkv.dim() != 2 or (qkv.shape[1] > 1 and qkv.stride(1) != 1) or qkv.shape[1] % dim:
        raise ValueError(f"qkv is [tokens, (heads + 2 kv_heads) * {dim}] of the pages' type with contiguous rows")
    heads = qkv.shape[1] // dim - 2 * kv
    if heads <= 0:
        raise ValueError(f"qkv of {qkv.shape[1]} columns has no query heads beside {kv} key and value heads of {dim}")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype is not torch.float32 or t.dim() != 2 or not t.is_contiguous() or t.shape != cos.shape:
            raise ValueError(f"{name} is a contiguous fp32 table [positions, rotary / 2], both alike")
    if out is None:
        out = torch.empty((qkv.shape[0], heads, dim), dtype=qkv.dtype, device=qkv.device)
    elif out.dtype is not qkv.dtype or out.shape != (qkv.shape[0], heads, dim) or not out.is_contiguous():
        raise ValueError(f"out is a contiguous [tokens, {heads}, {dim}] of qkv's type")
    _same_device(qkv.device, k_pages=k_pages, v_pages=v_pages, page_table=page_table, lengths=lengths, starts=starts, cos=cos, sin=sin,
                 positions=positions, out=out)
    stride = qkv.stride(0) if qkv.shape[0] > 1 else qkv.shape[1]
    with _on(qkv.device):
        _lib.check(_lib.lib().b200_paged_rope_append(
            ctypes.byref(cache), qkv.data_ptr(), stride, heads, cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1],
            int(interleaved), _index("positions", positions, (qkv.shape[0],)), out.data_ptr(), _stream_ptr(qkv.device)))
    return out


_scratch: dict = {}     # (device, stream) -> memory of paged_attention calls on that stream


def paged_attention_scratch(device) -> torch.Tensor:
    """Memory (79 MB) that paged_attention calls of one stream may share (``scratch=``): where several streams or captured graphs make
    such calls at the same time, each needs its own.  A call without it takes the stream's, which is kept; in a captured graph each takes
    and zeroes its own: one for the graph saves that."""
    with _on(device):
        size = int(_lib.lib().b200_paged_attention_scratch_bytes())
        if size < 0:
            _lib.check(_lib.ENODEVICE)
        scratch = torch.empty((size,), dtype=torch.uint8, device=device)
        scratch[:_lib.PAGED_ZEROED_BYTES].zero_()
    return scratch


def _stream_scratch(device) -> torch.Tensor:
    if torch._C._cuda_isCurrentStreamCapturing():       # a graph may be replayed beside anything: it has memory of its own
        return paged_attention_scratch(device)
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
    found = _scratch.get(key)
    if found is None:
        found = _scratch[key] = paged_attention_scratch(device)
    return found


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    starts: torch.Tensor | None = None, max_query: int | None = None, scale: float | None = None, causal: bool = True,
                    window: int = 0, cap: float = 0.0, slopes: torch.Tensor | None = None, prefix: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the rows q [tokens, heads, head_dim] over the keys and values of their sequences in the pages.

    ``lengths``, ``starts`` and the rows of a sequence as in :func:`paged_rope_append`, which has stored their keys before;
    ``max_query``: no sequence has more rows (None: the number of tokens).  A row at position t sees key j where j < prefix[b], or j <= t and
    (``window`` = 0 or t - j < window); ``causal`` = False: every key of its sequence.  Scores are scale * q.k (scale: 1 / sqrt(head_dim)),
    with ``cap`` > 0 cap * tanh(score / cap), with ``slopes`` (fp32 [heads]) less slopes[h] * |t - j|.  A row that sees nothing gets zeros.
    ``scratch``: see :func:`paged_attention_scratch`; None takes memory that belongs to the current stream."""
    native = _native or _torch_call()
    if native and q.is_cuda and torch._C._cuda_getDevice() == q.device.index:
        if scratch is None:
            scratch = _stream_scratch(q.device)
        result = native.paged_attention(q, k_pages, v_pages, page_table, lengths, starts, max_query, scale, causal, window, cap, slopes,
                                        prefix, out, scratch)
        if result is not None:
            return result
    cache = _paged_cache(q, k_pages, v_pages, page_table, lengths, starts, max_query)
    kv, dim = cache.kv_heads, cache.head_dim
    if q.dtype is not k_pages.dtype or q.dim() != 3 or q.shape[2] != dim or (q.shape[0] and (q.stride(2) != 1 or (q.shape[1] > 1 and q.stride(1) != dim))):
        raise ValueError(f"q is [tokens, heads, {dim}] of the pages' type, a token's heads contiguous")
    heads = q.shape[1]
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (heads,) or not slopes.is_contiguous()):
        raise ValueError(f"slopes are a contiguous fp32 tensor of {heads} values")
    if out is None:
        out = torch.empty((q.shape[0], heads, dim), dtype=q.dtype, device=q.device)
    elif out.dtype is not q.dtype or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out is a contiguous tensor of q's shape and type")
    if window < 0:
        raise ValueError(f"window is the number of tokens that a row sees, or 0: got {window}")
    _same_device(q.device, k_pages=k_pages, v_pages=v_pages, page_table=page_table, lengths=lengths, starts=starts, slopes=slopes,
                 prefix=prefix, out=out, scratch=scratch)
    with _on(q.device):
        if scratch is None:
            scratch = _stream_scratch(q.device)
        args = _lib.PagedAttention(q.data_ptr(), q.stride(0) if q.shape[0] > 1 else heads * dim, out.data_ptr(), heads, int(causal), min(int(window), 2 ** 31 - 1),
                                   dim ** -0.5 if scale is None else scale, cap, None if slopes is None else slopes.data_ptr(),
                                   _index("prefix", prefix, (cache.batch,)))
        _lib.check(_lib.lib().b200_paged_attention(ctypes.byref(cache), ctypes.byref(args), scratch.data_ptr(),
                                                   scratch.numel() * scratch.element_size(), _stream_ptr(q.device)))
    return out


class TokenLogprobs(typing.NamedTuple):
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor | None
    top_token: torch.Tensor | None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Of every row of logits [rows, V] (fp16, bf16 or fp32): the log probability of tokens[row] (int32), the entropy of the
    distribution and its ``top`` likeliest entries (at most 32; equal ones by index), all in fp32.  A logit of -inf is an excluded entry."""
    native = _native or _torch_call()
    if native:
        found = native.token_logprobs(logits, tokens, top)
        if found is not None:
            return TokenLogprobs(*found)
    if logits.dtype not in _LOGIT_TYPES or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits are an fp16, bf16 or fp32 tensor [rows, V] with contiguous rows")
    rows, V = logits.shape
    at = _index("tokens", tokens, (rows,))
    _same_device(logits.device, tokens=tokens)
    fp32 = dict(dtype=torch.float32, device=logits.device)
    logprob, entropy = torch.empty(rows, **fp32), torch.empty(rows, **fp32)
    best = torch.empty((rows, top), **fp32) if top else None
    best_token = torch.empty((rows, top), dtype=torch.int32, device=logits.device) if top else None
    with _on(logits.device):
        _lib.check(_lib.lib().b200_token_logprobs(
            logits.data_ptr(), _LOGIT_TYPES[logits.dtype], logits.stride(0) if rows > 1 else V, at, logprob.data_ptr(), entropy.data_ptr(),
            best.data_ptr() if top else None, best_token.data_ptr() if top else None, rows, V, top, _stream_ptr(logits.device)))
    return TokenLogprobs(logprob, entropy, best, best_token)


def launch_count() -> int:
    return int(_lib.lib().b200_launch_count())


def reset_launch_count() -> None:
    _lib.lib().b200_reset_launch_count()
