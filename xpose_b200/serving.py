"""Serving many sequences over one paged cache, on torch tensors.

Rotary positions (``rope_rows``), the quantising cache write and its read
(``kv_write``, ``kv_read``) and attention over whole prompts
(``attention_packed``) or of new tokens over the pages (``attention_paged``):
the ``xp_*`` calls of the same names in include/xp_cuda.h, whose comments give
the exact rules. Every call is enqueued on torch's current stream of the
tensors' device, which is one for all of them, and allocates nothing; errors
raise XpError. What only the device can see, a length past its table or a wait
that ran out, is in the scratch's error word: read it (error_word) where a
program waits for its results anyway.

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

from ._lib import XpError, check, lib

lib()  # the shared object loads, or fails loudly, before the binding that links to it
from . import _serving as _call  # noqa: E402

SCRATCH_BYTES = 48 << 20  # XP_SERVING_SCRATCH_BYTES

_LAYOUT = {"half": 0, "interleaved": 1}
_STRETCH = {"none": 0, "linear": 1, "base": 2, "parts": 3}


def _bad(message):
    return XpError(-1, message)


def _layout(name):
    if name not in _LAYOUT:
        raise _bad(f"layout must be 'half' or 'interleaved' (got {name!r})")
    return _LAYOUT[name]


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
    e = _call.rope_rows(out, x, positions, turns, _layout(layout), magnitude, inverse)
    if e is not None:
        raise XpError(*e)
    return out


def kv_write(k_pages, v_pages, k_scale, v_scale, k, v, slots, positions=None, turns=None, layout="half",
             magnitude=1.0):
    """k and v rows into the cache rows `slots`, k rotated first where turns are given."""
    e = _call.kv_write(k_pages, v_pages, k_scale, v_scale, k, v, slots, positions, turns, _layout(layout), magnitude)
    if e is not None:
        raise XpError(*e)


def kv_read(k_pages, v_pages, k_scale, v_scale, k, v, slots):
    """The cache rows `slots` as values into k and v."""
    e = _call.kv_read(k_pages, v_pages, k_scale, v_scale, k, v, slots)
    if e is not None:
        raise XpError(*e)


def attention_packed(out, q, k, v, starts, scratch, window=0, scale=0.0, lse=None):
    """Causal attention over whole prompts: sequence b is tokens starts[b] .. starts[b + 1] - 1."""
    e = _call.attention_packed(out, q, k, v, starts, scratch, window, scale, lse)
    if e is not None:
        raise XpError(*e)
    return out


def attention_paged(out, q, k_pages, v_pages, k_scale, v_scale, table, kv_lens, starts, q_most, scratch, window=0,
                    scale=0.0, lse=None):
    """Attention of each sequence's new tokens (q rows starts[b] .. starts[b + 1] - 1) over its kv_lens[b] keys in
    pages table[b]; q_most is the most new tokens of any sequence."""
    e = _call.attention_paged(out, q, k_pages, v_pages, k_scale, v_scale, table, kv_lens, starts, q_most, scratch,
                              window, scale, lse)
    if e is not None:
        raise XpError(*e)
    return out
