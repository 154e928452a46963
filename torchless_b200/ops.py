"""Device ops with the names and argument order of src/common/kernels.h.

Each function takes CUDA float32 tensors (int8 for quantised weights) and
launches on torch's current stream.  Output first, like the reference:
``matmul(xout, w, x)`` computes ``xout = w @ x``.  Shapes follow the
reference's Tensor shapes; in-place calls (``xout is x``) are allowed where
the reference makes them (rope, softmax, silu, mul in modules.cpp).
"""
from __future__ import annotations

import ctypes

from . import check, lib, tl_paged_cache


def _ptr(t) -> int:
    if not t.is_cuda:
        raise ValueError("ops take CUDA tensors")
    if not t.is_contiguous():
        raise ValueError("ops take contiguous tensors")
    return t.data_ptr()


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _f32(t):
    import torch
    if t.dtype != torch.float32:
        raise TypeError(f"expected float32, got {t.dtype}")
    return _ptr(t)


def matmul(xout, w, x, scales=None) -> None:
    """kernels.h:11-12: xout[n] = w[n, d] @ x[d]; int8 ``w`` needs its stored
    ``scales``; fp8 ``w`` (torch.float8_e5m2, or uint8 holding e5m2 bit
    patterns: the fp8 export) has none."""
    import torch
    n, d = w.shape
    if x.numel() != d or xout.numel() < n:
        raise ValueError("matmul shape mismatch")  # kernels.cpp:10, 25
    if w.dtype in (torch.float8_e5m2, torch.uint8):
        if scales is not None:
            raise ValueError("fp8 weights have no scales")
        check(lib().tl_matmul_f8(_f32(xout), _ptr(w), _f32(x), n, d, _stream()))
    elif w.dtype == torch.int8:
        if scales is None:
            raise ValueError("int8 matmul needs scales")
        check(lib().tl_matmul_i8(_f32(xout), _ptr(w), _f32(scales), scales.numel(), _f32(x), n, d, _stream()))
    else:
        check(lib().tl_matmul_f32(_f32(xout), _f32(w), _f32(x), n, d, _stream()))


def row_matmul(xout, x, w) -> None:
    """kernels.h:13: xout[d] = x[n] @ w[n, d]."""
    n, d = w.shape
    if x.shape[0] != n or xout.numel() < d:
        raise ValueError("matmul shape mismatch")  # kernels.cpp:42
    check(lib().tl_row_matmul(_f32(xout), _f32(x), _f32(w), n, d, _stream()))


def softmax(xout, x) -> None:
    check(lib().tl_softmax(_f32(xout), _f32(x), x.numel(), _stream()))


def rope(xout, x, cos, sin) -> None:
    """kernels.h:16: x is [n_heads, head_dim]."""
    n_heads, head_dim = x.shape
    check(lib().tl_rope(_f32(xout), _f32(x), _f32(cos), _f32(sin), n_heads, head_dim, _stream()))


def silu(xout, x) -> None:
    check(lib().tl_silu(_f32(xout), _f32(x), x.numel(), _stream()))


def sum(x):
    """kernels.h:20: returns a 1-element device tensor."""
    import torch
    out = torch.empty(1, dtype=torch.float32, device=x.device)
    check(lib().tl_sum(_f32(out), _f32(x), x.numel(), _stream()))
    return out


def add(xout, x, y) -> None:
    if isinstance(y, (int, float)):
        check(lib().tl_add_scalar(_f32(xout), _f32(x), float(y), x.numel(), _stream()))
    else:
        check(lib().tl_add(_f32(xout), _f32(x), _f32(y), x.numel(), _stream()))


def mul(xout, x, y) -> None:
    if isinstance(y, (int, float)):
        check(lib().tl_mul_scalar(_f32(xout), _f32(x), float(y), x.numel(), _stream()))
    else:
        check(lib().tl_mul(_f32(xout), _f32(x), _f32(y), x.numel(), _stream()))


def pow(xout, x, e: int) -> None:  # noqa: A001 - reference name
    check(lib().tl_pow(_f32(xout), _f32(x), int(e), x.numel(), _stream()))


def sqrt(xout, x) -> None:
    check(lib().tl_sqrt(_f32(xout), _f32(x), x.numel(), _stream()))


def rmsnorm(xout, x, g, eps: float = 1e-5) -> None:
    """RMSNorm::forward (modules.cpp:31-46)."""
    check(lib().tl_rmsnorm(_f32(xout), _f32(x), _f32(g), x.numel(), float(eps), _stream()))


def rotary(cos, sin, inv_freq, pos: int) -> None:
    """RotaryEmbedding::forward (modules.cpp:22-27)."""
    check(lib().tl_rotary(_f32(cos), _f32(sin), _f32(inv_freq), inv_freq.numel(), cos.numel(), int(pos),
                          _stream()))


def argmax(logits):
    """sample_max (main.cpp:10-21); returns a 1-element uint32 device tensor (as int32)."""
    import torch
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(lib().tl_argmax(_ptr(out), _f32(logits), logits.numel(), _stream()))
    return out


def sample_multinomial(logits, temperature: float, r: float):
    """sample_multinomial (main.cpp:23-43) with the uniform draw r given; returns a
    1-element device tensor (int32) holding the index."""
    import torch
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    check(lib().tl_sample_multinomial(_ptr(out), _f32(logits), logits.numel(), float(temperature), float(r),
                                      _stream()))
    return out


def sample_uniform(seed: int, pos: int) -> float:
    """The uniform draw of device-side sampling for the token at position pos."""
    return float(lib().tl_sample_uniform(int(seed), int(pos)))


def mlp_gate_up(out, w1, s1, w3, s3, x) -> None:
    """silu(w1 @ x) * (w3 @ x) with int8 w1/w3 (modules.cpp:99-112)."""
    n, d = w1.shape
    check(lib().tl_mlp_gate_up(_f32(out), _ptr(w1), _f32(s1), _ptr(w3), _f32(s3), _f32(x), n, d, _stream()))


def quantize_i8(x, group: int = 64):
    """quantize (export_mistral.py:53-68) on the device: returns (q int8, scales f32)."""
    import torch
    xc = x.contiguous()
    q = torch.empty(xc.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(xc.numel() // group, dtype=torch.float32, device=x.device)
    check(lib().tl_quantize_i8(_ptr(q), _f32(s), _f32(xc), xc.numel(), group, _stream()))
    return q, s


# ---- serving step over a paged KV cache (no reference counterpart: its
# InferenceState, inference_state.h:8-72, holds one sequence) ----
#
# The pages of a layer are two tensors k_cache, v_cache
# [n_blocks, n_kv_heads, block_size, head_dim] (float32, float16 or bfloat16),
# contiguous but for the stride between pages.  Lengths, tables and settings
# of requests are int32 / float32 tensors on the device, never read by the
# host, so a step can be captured in a CUDA graph.


_torch = None   # torch, from the first call on
_DTYPES = {}    # the cache's types by torch's


def _load():
    global _torch
    import torch
    _DTYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    _torch = torch
    return torch


def _launch(index, f, *args) -> None:
    """f(*args, current stream of device `index`), with that device current."""
    C = _torch._C
    stream = C._cuda_getCurrentRawStream(index)
    before = C._cuda_getDevice()
    if before == index:
        st = f(*args, stream)
    else:
        _torch.cuda.set_device(index)
        try:
            st = f(*args, stream)
        finally:
            _torch.cuda.set_device(before)
    if st:
        check(st)


def _dtype(t) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"expected float32, float16 or bfloat16, got {t.dtype}") from None


def _arg(t, dtype, index, n, name):
    """A contiguous tensor of `dtype` on device `index` with n elements (None: any): its address."""
    if t.dtype is dtype and t.get_device() == index and t.is_contiguous() and (n is None or t.numel() == n):
        return t.data_ptr()
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not cuda:{index}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    raise ValueError(f"{name} has {t.numel()} elements, not {n}")


def _cache(k_cache, v_cache):
    """The pages as the library's structure, and their device."""
    shape, st, sv, index = k_cache.shape, k_cache.stride(), v_cache.stride(), k_cache.get_device()
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [n_blocks, n_kv_heads, block_size, head_dim] of one layout")
    if index < 0 or v_cache.get_device() != index or k_cache.dtype is not v_cache.dtype:
        raise ValueError("k_cache and v_cache must be CUDA tensors of one type and device")
    n, kv, bs, hd = shape
    if n > 1 and st[0] != sv[0]:
        raise ValueError("k_cache and v_cache must be of one layout")
    inside = (bs * hd, hd, 1)
    if n and (st[1:] != inside or sv[1:] != inside) and not (k_cache[0].is_contiguous() and v_cache[0].is_contiguous()):
        raise ValueError("the pages of a cache must be contiguous")  # (a dimension of size 1 may have any stride)
    return tl_paged_cache(k_cache.data_ptr(), v_cache.data_ptr(), n, kv, bs, hd,
                          st[0] if n > 1 else kv * bs * hd, _dtype(k_cache)), index


def paged_plan(block_table, cached, new_tokens, free_blocks, block_size: int, n_tokens: int):
    """Block tables and slot maps of a step from the request lengths.

    ``block_table`` [n_req, max_blocks] is extended in place by the pages that
    the new tokens need, taken from ``free_blocks`` in order (-1 once it is used
    up).  ``cached`` and ``new_tokens`` [n_req] are each request's tokens
    before and in this step; the new tokens lie one after the other in
    ``n_tokens`` rows.  Returns int32 tensors
    ``(q_start [n_req + 1], seq_lens [n_req], positions [n_tokens],
    slots [n_tokens], counts [2])``; position and slot are -1 in rows behind
    the last token, the slot of a token without a page is -1, and counts are
    the pages taken and the pages missing."""
    torch = _torch or _load()
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_req, max_blocks]")
    n_req, width = block_table.shape
    index, i32 = block_table.get_device(), torch.int32
    if index < 0:
        raise ValueError("ops take CUDA tensors")
    if n_tokens < 0 or block_size < 0:
        raise ValueError("n_tokens and block_size must not be negative")
    table, before, new, free = (
        _arg(block_table, i32, index, None, "block_table"), _arg(cached, i32, index, n_req, "cached"),
        _arg(new_tokens, i32, index, n_req, "new_tokens"), _arg(free_blocks, i32, index, None, "free_blocks"))
    out = torch.empty(2 * n_req + 2 * n_tokens + 3, dtype=i32, device=block_table.device)
    q_start = out.data_ptr()
    seq_lens = q_start + 4 * (n_req + 1)
    positions = seq_lens + 4 * n_req
    slots = positions + 4 * n_tokens
    _launch(index, lib().tl_paged_plan, table, q_start, seq_lens, positions, slots, slots + 4 * n_tokens, before, new, free,
            free_blocks.numel(), n_req, width, block_size, n_tokens)
    return out.split_with_sizes((n_req + 1, n_req, n_tokens, n_tokens, 2))


def qk_norm_rope(q_out, k_cache, v_cache, qkv, positions, slots, cos, sin, q_weight=None, k_weight=None,
                 eps: float = 1e-5) -> None:
    """RMSNorm of each q and k head (where its weight is given), rotation and
    the write of k and v into their pages, in one pass.

    ``qkv`` [n_tokens, (n_heads + 2 n_kv_heads) * head_dim] (rows may be
    strided), ``q_out`` [n_tokens, n_heads, head_dim] in the cache's type,
    ``positions`` / ``slots`` as paged_plan gives them, ``cos`` / ``sin``
    float32 [n_pos, rot_dim / 2].  Rows with a position outside the tables are
    left alone; rows without a page get their q only."""
    torch = _torch or _load()
    c, index = _cache(k_cache, v_cache)
    i32, f32 = torch.int32, torch.float32
    if q_out.dim() != 3 or q_out.dtype is not k_cache.dtype:
        raise ValueError("q_out must be [n_tokens, n_heads, head_dim] in the cache's type")
    n, heads, hd = q_out.shape
    if hd != c.head_dim:
        raise ValueError("q_out must be [n_tokens, n_heads, head_dim] in the cache's type")
    if qkv.shape != (n, (heads + 2 * c.n_kv_heads) * hd):
        raise ValueError("qkv must be [n_tokens, (n_heads + 2 n_kv_heads) * head_dim]")
    stride, one = qkv.stride()
    if n and one != 1:
        raise ValueError("the heads of a token must be contiguous in qkv")
    if qkv.get_device() != index:
        raise ValueError(f"qkv is on {qkv.device}, not cuda:{index}")
    if cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError("cos and sin must be [n_pos, rot_dim / 2]")
    n_pos, half = cos.shape
    _launch(index, lib().tl_qk_norm_rope, _arg(q_out, q_out.dtype, index, None, "q_out"), ctypes.byref(c), qkv.data_ptr(),
            _dtype(qkv), stride if n > 1 else (heads + 2 * c.n_kv_heads) * hd, _arg(positions, i32, index, n, "positions"),
            _arg(slots, i32, index, n, "slots"), _arg(cos, f32, index, None, "cos"), _arg(sin, f32, index, None, "sin"),
            n_pos, 2 * half, None if q_weight is None else _arg(q_weight, f32, index, hd, "q_weight"),
            None if k_weight is None else _arg(k_weight, f32, index, hd, "k_weight"), eps, n, heads)


def paged_attention(out, q, k_cache, v_cache, block_table, q_start, seq_lens, scale=None, window: int = 0) -> None:
    """Causal GQA attention of each sequence's new tokens over its pages.

    ``q`` and ``out`` [n_tokens, n_heads, head_dim] in the cache's type (``q``
    may be strided between tokens); sequence b has the rows q_start[b] ..
    q_start[b + 1), which are the last of its seq_lens[b] tokens.  ``scale``
    defaults to 1 / sqrt(head_dim); ``window`` > 0 attends to that many last
    positions.  A query that attends to nothing gets zeros; rows of no sequence
    are left as they were."""
    torch = _torch or _load()
    c, index = _cache(k_cache, v_cache)
    i32, dtype = torch.int32, q.dtype
    if q.dim() != 3 or dtype is not k_cache.dtype or q.shape != out.shape:
        raise ValueError("q and out must be [n_tokens, n_heads, head_dim] in the cache's type")
    n, heads, hd = q.shape
    stride, of_head, one = q.stride()
    if hd != c.head_dim or out.dtype is not dtype:
        raise ValueError("q and out must be [n_tokens, n_heads, head_dim] in the cache's type")
    if n and (one != 1 or (heads > 1 and of_head != hd)):
        raise ValueError("the heads of a token must be contiguous in q")
    if q.get_device() != index:
        raise ValueError(f"q is on {q.device}, not cuda:{index}")
    if block_table.dim() != 2 or window < 0:
        raise ValueError("block_table must be [n_seq, max_blocks] and window not negative")
    n_seq, width = block_table.shape
    L, cache = lib(), ctypes.byref(c)
    key = (index, c.dtype, hd, c.n_kv_heads, heads, n, n_seq)
    need = _WORKSPACE.get(key)
    if need is None:
        size = ctypes.c_size_t()
        with torch.cuda.device(index):
            check(L.tl_paged_attention_workspace(cache, n, heads, n_seq, width, ctypes.byref(size)))
        if len(_WORKSPACE) >= 4096:
            _WORKSPACE.clear()
        need = _WORKSPACE[key] = size.value
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    _launch(index, L.tl_paged_attention, _arg(out, dtype, index, None, "out"), q.data_ptr(),
            stride if n > 1 else heads * hd, cache, _arg(block_table, i32, index, None, "block_table"), width,
            _arg(q_start, i32, index, n_seq + 1, "q_start"), _arg(seq_lens, i32, index, n_seq, "seq_lens"), n_seq, n, heads,
            hd ** -0.5 if scale is None else scale, window, ws.data_ptr(), need)


_WORKSPACE = {}  # the workspace's size by device, type, heads and numbers of rows and sequences


def sample_rows(logits, r, temperature, top_k=None, top_p=None, min_p=None):
    """sample_multinomial for each row of ``logits`` [n_rows, n] (float32,
    float16 or bfloat16; rows may be strided) with the row's own uniform draw
    ``r`` in [0, 1), ``temperature`` (<= 0: sample_max), and optionally
    ``top_k`` (int32; <= 0: off), ``top_p`` (>= 1: off) and ``min_p`` (<= 0:
    off; > 1: the largest alone), applied in that order.  Returns the indexes, an int32 tensor [n_rows]."""
    torch = _torch or _load()
    if logits.dim() != 2:
        raise ValueError("logits must be [n_rows, n] with contiguous rows")
    rows, n = logits.shape
    stride, one = logits.stride()
    if rows and n > 1 and one != 1:
        raise ValueError("logits must be [n_rows, n] with contiguous rows")
    index, f32, i32 = logits.get_device(), torch.float32, torch.int32
    if index < 0:
        raise ValueError("ops take CUDA tensors")
    draws, temps = _arg(r, f32, index, rows, "r"), _arg(temperature, f32, index, rows, "temperature")
    k = None if top_k is None else _arg(top_k, i32, index, rows, "top_k")
    p = None if top_p is None else _arg(top_p, f32, index, rows, "top_p")
    m = None if min_p is None else _arg(min_p, f32, index, rows, "min_p")
    out = torch.empty(rows, dtype=i32, device=logits.device)
    _launch(index, lib().tl_sample_rows, out.data_ptr(), logits.data_ptr(), _dtype(logits), stride if rows > 1 else n, rows, n,
            draws, temps, k, p, m)
    return out
