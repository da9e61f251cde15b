"""Serving many sequences over one paged cache, on torch tensors.

Rotary positions (``rope_rows``), the quantising cache write and its read
(``kv_write``, ``kv_read``) and attention over whole prompts
(``attention_packed``) or of new tokens over the pages (``attention_paged``):
the ``xp_*`` calls of the same names in include/xp_cuda.h, whose comments give
the exact rules. Every call is enqueued on torch's current stream of the
tensors' device and allocates nothing; errors raise XpError.

    turns, magnitude = rope_turns(256, 1e6)
    k_pages, v_pages, k_scale, v_scale = new_pages(1024, 16, 1, 256, torch.int8)
    scratch = new_scratch()
    rope_rows(q, q, positions, turns)
    kv_write(k_pages, v_pages, k_scale, v_scale, k, v, slots, positions=positions, turns=turns)
    attention_paged(out, q, k_pages, v_pages, k_scale, v_scale, table, kv_lens, starts, q_most, scratch)

Rows of heads are tensors [tokens, heads, dim] whose last axis is contiguous;
the other strides are free. Pages are contiguous [pages, kv heads, page size,
dim] of float16, bfloat16, int8 or float8_e4m3fn, the last two with float32
scales [pages, kv heads, page size].
"""
import ctypes as C

import torch

from ._lib import Pages, Rotary, Rows, XpError, check, lib

SCRATCH_BYTES = 48 << 20  # XP_SERVING_SCRATCH_BYTES

_ROWS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_PAGES = {torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_LAYOUT = {"half": 0, "interleaved": 1}
_STRETCH = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def _bad(message):
    return XpError(-1, message)


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _rows(name, t):
    if t.dim() != 3 or not t.is_cuda or t.dtype not in _ROWS:
        raise _bad(f"'{name}' must be a CUDA tensor [tokens, heads, dim] of float32, float16 or bfloat16")
    n, h, d = t.shape
    ts, hs, ds = t.stride()
    if ds != 1 and d > 1:
        raise _bad(f"the last axis of '{name}' must be contiguous")
    return Rows(t.data_ptr(), ts if n > 1 else 0, hs if h > 1 else 0, n, h, d, _ROWS[t.dtype])


def _pages(k, v, k_scale, v_scale):
    if k.dim() != 4 or not k.is_cuda or k.dtype not in _PAGES or v.dtype != k.dtype or v.shape != k.shape:
        raise _bad("the pages must be two CUDA tensors [pages, kv heads, page size, dim] of one cache type")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise _bad("the pages must be contiguous")
    n, h, p, d = k.shape
    ks = vs = None
    if k.element_size() == 1:
        for s in (k_scale, v_scale):
            if s is None or s.dtype != torch.float32 or s.shape != (n, h, p) or not s.is_contiguous():
                raise _bad("8-bit pages need contiguous float32 scales [pages, kv heads, page size]")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    return Pages(k.data_ptr(), v.data_ptr(), ks, vs, n, p, h, d, _PAGES[k.dtype])


def _ints(name, t, n, dtype):
    if t.dtype != dtype or not t.is_cuda or t.numel() != n or not t.is_contiguous():
        raise _bad(f"'{name}' must be a contiguous CUDA tensor of {n} {dtype}")
    return t.data_ptr()


def _rotary(rows, positions, turns, layout, magnitude, inverse):
    if layout not in _LAYOUT:
        raise _bad(f"layout must be 'half' or 'interleaved' (got {layout!r})")
    n = turns.numel()
    return Rotary(_ints("turns", turns, n, torch.int64), _ints("positions", positions, rows.tokens, torch.int32),
                  2 * n, _LAYOUT[layout], magnitude, inverse)


def rope_turns(rot_dim, theta, stretch="none", factor=1.0, original=8192, slow=1.0, fast=32.0, device="cuda"):
    """The frequency table of a rotary embedding, 64-bit fractions of a turn a
    position as int64 [rot_dim / 2], and the magnitude that goes with it."""
    if stretch not in _STRETCH:
        raise _bad(f"stretch must be one of {', '.join(_STRETCH)} (got {stretch!r})")
    buf, magnitude = (C.c_int64 * max(1, rot_dim // 2))(), C.c_float()
    check(lib().xp_rope_turns(buf, C.byref(magnitude), rot_dim, theta, _STRETCH[stretch], factor, original, slow, fast))
    return torch.tensor(list(buf), dtype=torch.int64, device=device), magnitude.value


def new_pages(pages, page_size, kv_heads, dim, dtype, device="cuda"):
    """(k, v, k_scale, v_scale) of an empty cache; the scales are None for 16-bit types."""
    shape = (pages, kv_heads, page_size, dim)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if dtype.itemsize == 1
            else torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype.itemsize > 1:
        return k, v, None, None
    return (k, v) + tuple(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))


def new_scratch(device="cuda"):
    """A workspace of the two attentions: one call at a time may use it."""
    return torch.zeros(SCRATCH_BYTES, dtype=torch.uint8, device=device)


def error_word(scratch, clear=True):
    """The workspace's sticky error word (see XP_SERVING_SCRATCH_BYTES); waits for the stream."""
    word = scratch[4:8].view(torch.int32)
    value = int(word.item())
    if clear:
        word.zero_()
    return value


def rope_rows(out, x, positions, turns, layout="half", magnitude=1.0, inverse=False):
    """out = x with every head rotated to its token's position; out may be x."""
    a, b = _rows("out", out), _rows("x", x)
    r = _rotary(b, positions, turns, layout, magnitude, inverse)
    check(lib().xp_rope_rows(_stream(x), C.byref(a), C.byref(b), C.byref(r)))
    return out


def kv_write(k_pages, v_pages, k_scale, v_scale, k, v, slots, positions=None, turns=None, layout="half",
             magnitude=1.0):
    """k and v rows into the cache rows `slots`, k rotated first where turns are given."""
    p, a, b = _pages(k_pages, v_pages, k_scale, v_scale), _rows("k", k), _rows("v", v)
    r = None if turns is None else C.byref(_rotary(a, positions, turns, layout, magnitude, False))
    check(lib().xp_kv_write(_stream(k), C.byref(p), C.byref(a), C.byref(b),
                            _ints("slots", slots, a.tokens, torch.int64), r))


def kv_read(k_pages, v_pages, k_scale, v_scale, k, v, slots):
    """The cache rows `slots` as values into k and v."""
    p, a, b = _pages(k_pages, v_pages, k_scale, v_scale), _rows("k", k), _rows("v", v)
    check(lib().xp_kv_read(_stream(k), C.byref(p), C.byref(a), C.byref(b),
                           _ints("slots", slots, a.tokens, torch.int64)))


def _scratch(t):
    if not t.is_cuda or t.numel() * t.element_size() < SCRATCH_BYTES:
        raise _bad(f"'scratch' must be a CUDA tensor of {SCRATCH_BYTES} bytes (new_scratch)")
    return t.data_ptr()


def _lse(lse, q):
    if lse is None:
        return None
    return _ints("lse", lse, q.tokens * q.heads, torch.float32)


def attention_packed(out, q, k, v, starts, scratch, window=0, scale=0.0, lse=None):
    """Causal attention over whole prompts: sequence b is tokens starts[b] .. starts[b + 1] - 1."""
    o, a, b, c = _rows("out", out), _rows("q", q), _rows("k", k), _rows("v", v)
    n = starts.numel() - 1
    check(lib().xp_attention_packed(_stream(q), C.byref(o), C.byref(a), C.byref(b), C.byref(c),
                                    _ints("starts", starts, n + 1, torch.int32), n, window, scale, _lse(lse, a),
                                    _scratch(scratch)))
    return out


def attention_paged(out, q, k_pages, v_pages, k_scale, v_scale, table, kv_lens, starts, q_most, scratch, window=0,
                    scale=0.0, lse=None):
    """Attention of each sequence's new tokens (q rows starts[b] .. starts[b + 1] - 1) over its kv_lens[b] keys in
    pages table[b]; q_most is the most new tokens of any sequence."""
    o, a, p = _rows("out", out), _rows("q", q), _pages(k_pages, v_pages, k_scale, v_scale)
    n = kv_lens.numel()
    if table.dim() != 2 or table.shape[0] != n:
        raise _bad("'table' must be [sequences, pages of a sequence]")
    width = table.shape[1]
    check(lib().xp_attention_paged(_stream(q), C.byref(o), C.byref(a), C.byref(p),
                                   _ints("table", table, n * width, torch.int32), width,
                                   _ints("kv_lens", kv_lens, n, torch.int32),
                                   _ints("starts", starts, n + 1, torch.int32), n, q_most, window, scale,
                                   _lse(lse, a), _scratch(scratch)))
    return out
