"""The serving operators' host side without a GPU: the frequency tables
against Python's arithmetic, and what the C entry points refuse before they
touch a device."""
import ctypes as C
import math

import pytest

from xpose_b200._lib import Pages, Rotary, Rows, XpError, check, lib

F32, F16, BF16, I8, FP8 = range(5)
P = 1 << 20  # a non-null, aligned pointer value: nothing reads it


def turns(rot, theta, stretch=0, factor=1.0, original=8192.0, slow=1.0, fast=32.0):
    buf, m = (C.c_uint64 * max(1, rot // 2))(), C.c_float()
    check(lib().xp_rope_turns(buf, C.byref(m), rot, theta, stretch, factor, original, slow, fast))
    return list(buf), m.value


@pytest.mark.parametrize("rot,theta", [(2, 1e4), (64, 1e4), (128, 5e5), (256, 1e6), (6, 1.5)])
@pytest.mark.parametrize("stretch,factor", [(0, 1.0), (1, 8.0), (2, 4.0), (3, 32.0)])
def test_rope_turns(rot, theta, stretch, factor):
    if stretch == 2 and rot == 2:
        with pytest.raises(XpError):
            turns(rot, theta, stretch, factor)
        return
    got, m = turns(rot, theta, stretch, factor)
    base = theta * factor ** (rot / (rot - 2)) if stretch == 2 else theta
    for i, t in enumerate(got):
        f = base ** (-2.0 * i / rot)
        if stretch == 1:
            f /= factor
        if stretch == 3:
            g = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1.0) / 31.0))
            f *= g + (1 - g) / factor
        # a step of the table (2^-64 of a turn), and a few roundings of a double (2^-53) in pow
        assert abs(t / 2.0 ** 64 - f / (2 * math.pi)) <= 2.0 ** -64 + 2.0 ** -49 * f / (2 * math.pi)
    assert m == pytest.approx(0.1 * math.log(factor) + 1 if stretch == 3 else 1.0)


@pytest.mark.parametrize("args", [(0, 1e4), (7, 1e4), (64, 1.0), (64, math.inf), (64, 1e4, 4), (64, 1e4, 1, 0.5),
                                  (64, 1e4, 3, 2.0, 0.0), (64, 1e4, 3, 2.0, 8192.0, 4.0, 4.0)])
def test_rope_turns_refuses(args):
    with pytest.raises(XpError) as e:
        turns(*args)
    assert e.value.name == "XP_ERR_INVALID" and "rope_turns" in str(e.value)


def rows(tokens=4, heads=4, dim=128, dtype=F16, data=P, ts=None, hs=None):
    return Rows(data, heads * dim if ts is None else ts, dim if hs is None else hs, tokens, heads, dim, dtype)


def pages(dtype=I8, page=16, kv=1, dim=128, n=8, k=P, ks=P):
    return Pages(k, P, ks, P, n, page, kv, dim, dtype)


def rotary(rot=128, layout=0, t=P, pos=P):
    return Rotary(t, pos, rot, layout, 1.0, 0)


def refused(status, *words):
    message = lib().xp_last_error().decode()
    assert status == -1, (status, message)
    for w in words:
        assert w in message, message


def ref(x):
    return None if x is None else C.byref(x)


@pytest.mark.parametrize("out,x,r,word", [
    (None, rows(), rotary(), "'out'"), (rows(), None, rotary(), "'in'"), (rows(), rows(), None, "'rope'"),
    (rows(heads=2), rows(), rotary(), "shape"), (rows(dtype=BF16), rows(), rotary(), "type"),
    (rows(), rows(), rotary(rot=130), "rot_dim"), (rows(), rows(), rotary(rot=7), "rot_dim"),
    (rows(), rows(), rotary(rot=0), "rot_dim"), (rows(), rows(), rotary(layout=2), "layout"),
    (rows(), rows(), rotary(t=None), "turns"), (rows(dtype=I8), rows(dtype=I8), rotary(), "F32"),
    (rows(data=None), rows(), rotary(), "no data"), (rows(), rows(data=P + 1), rotary(), "aligned")])
def test_rope_rows_refuses(out, x, r, word):
    refused(lib().xp_rope_rows(None, ref(out), ref(x), ref(r)), "rope_rows", word)


@pytest.mark.parametrize("p,k,v,slots,r,word", [
    (None, rows(heads=1), rows(heads=1), P, None, "'pages'"), (pages(), None, rows(heads=1), P, None, "'k'"),
    (pages(page=24), rows(heads=1), rows(heads=1), P, None, "page_size"),
    (pages(page=4), rows(heads=1), rows(heads=1), P, None, "page_size"),
    (pages(page=512), rows(heads=1), rows(heads=1), P, None, "page_size"),
    (pages(dim=96), rows(heads=1, dim=96), rows(heads=1, dim=96), P, None, "head_dim"),
    (pages(dtype=F32), rows(heads=1), rows(heads=1), P, None, "INT8"),
    (pages(ks=None), rows(heads=1), rows(heads=1), P, None, "scales"),
    (pages(k=P + 8), rows(heads=1), rows(heads=1), P, None, "aligned"),
    (pages(n=0), rows(heads=1), rows(heads=1), P, None, "empty"),
    (pages(), rows(heads=2), rows(heads=2), P, None, "shape"),
    (pages(), rows(heads=1), rows(heads=1, tokens=3), P, None, "shape"),
    (pages(), rows(heads=1), rows(heads=1, data=P + 2), P, None, "aligned"),
    (pages(), rows(heads=1), rows(heads=1), None, None, "'slots'"),
    (pages(), rows(heads=1), rows(heads=1), P, rotary(rot=130), "rot_dim"),
    (pages(), rows(heads=1), rows(heads=1), P, rotary(rot=6), "rot_dim")])
def test_kv_refuses(p, k, v, slots, r, word):
    refused(lib().xp_kv_write(None, ref(p), ref(k), ref(v), slots, ref(r)), "kv_write", word)
    if r is None:
        refused(lib().xp_kv_read(None, ref(p), ref(k), ref(v), slots), "kv_read", word)


def packed(out=None, q=None, k=None, v=None, starts=P, scale=0.0, scratch=P):
    return lib().xp_attention_packed(None, ref(out or rows()), ref(q or rows()), ref(k or rows(heads=1)),
                                     ref(v or rows(heads=1)), starts, 2, 0, scale, None, scratch)


@pytest.mark.parametrize("kw,word", [
    (dict(q=rows(dim=96), out=rows(dim=96)), "dim"), (dict(q=rows(dtype=F32), out=rows(dtype=F32)), "F16 or BF16"),
    (dict(out=rows(heads=2)), "'out'"), (dict(k=rows(heads=3), v=rows(heads=3)), "kv heads"),
    (dict(k=rows(heads=1, dtype=BF16)), "differ"), (dict(v=rows(heads=2)), "differ"),
    (dict(k=rows(heads=1, tokens=3), v=rows(heads=1, tokens=3)), "differ"),
    (dict(q=rows(ts=516)), "aligned"), (dict(q=rows(data=P + 8)), "aligned"), (dict(starts=None), "'starts'"),
    (dict(scratch=None), "'scratch'"), (dict(scratch=P + 4), "'scratch'"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale")])
def test_attention_packed_refuses(kw, word):
    refused(packed(**kw), "attention_packed", word)


def paged(out=None, q=None, p=None, table=P, width=4, kv_lens=P, starts=P, scratch=P):
    return lib().xp_attention_paged(None, ref(out or rows()), ref(q or rows()), ref(p or pages()), table, width,
                                    kv_lens, starts, 2, 1, 0, 0.0, None, scratch)


@pytest.mark.parametrize("kw,word", [
    (dict(p=pages(dim=64)), "dim"), (dict(p=pages(dtype=BF16)), "type"), (dict(p=pages(kv=3)), "kv heads"),
    (dict(table=None), "'table'"), (dict(kv_lens=None), "'kv_lens'"), (dict(starts=None), "'starts'"),
    (dict(width=1 << 27), "2^31"), (dict(scratch=None), "'scratch'")])
def test_attention_paged_refuses(kw, word):
    refused(paged(**kw), "attention_paged", word)


def test_attention_paged_refuses_no_pages():
    refused(lib().xp_attention_paged(None, ref(rows()), ref(rows()), None, P, 1, P, P, 1, 1, 0, 0.0, None, P), "'pages'")


# rows that overlap: one for all, a stride below the head's size, or both axes together
OVERLAP = [dict(ts=0), dict(hs=0), dict(ts=64), dict(hs=64), dict(hs=-64), dict(ts=128, hs=256, heads=2),
           dict(ts=384, hs=512, heads=4, tokens=5), dict(ts=3 * 128, hs=-2 * 128 - 64, heads=4, tokens=9)]


@pytest.mark.parametrize("layout", OVERLAP)
def test_rows_that_are_written_must_not_overlap(layout):
    x = {"heads": 4, "tokens": 4} | layout
    good, bad = rows(heads=x["heads"], tokens=x["tokens"]), rows(**x)
    refused(lib().xp_rope_rows(None, ref(bad), ref(good), ref(rotary())), "rope_rows", "'out' overlap")
    p = pages(kv=x["heads"])
    refused(lib().xp_kv_read(None, ref(p), ref(bad), ref(good), P), "kv_read", "'k' overlap")
    refused(lib().xp_kv_read(None, ref(p), ref(good), ref(bad), P), "kv_read", "'v' overlap")
    one = rows(heads=1, tokens=x["tokens"])
    refused(packed(out=bad, q=good, k=one, v=one), "attention_packed", "'out' overlap")
    refused(paged(out=bad, q=good), "attention_paged", "'out' overlap")


@pytest.mark.parametrize("layout", [dict(ts=1024), dict(hs=256, ts=1024), dict(ts=128, hs=512)])
def test_rope_rows_in_place_keeps_its_strides(layout):
    """Rows of one place in two orders: a thread would read what another has written."""
    refused(lib().xp_rope_rows(None, ref(rows(**layout)), ref(rows()), ref(rotary())), "rope_rows", "strides")
