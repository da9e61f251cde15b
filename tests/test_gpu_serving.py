"""The serving operators (xpose_b200.serving) against plain 64-bit forms."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import serving_ref as R  # noqa: E402
from xpose_b200 import serving as S  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I8, FP8 = torch.int8, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def starts_of(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return ints(at)


@pytest.fixture(scope="module")
def scratch():
    return S.new_scratch()


# ---- rotary rows ------------------------------------------------------------
def freqs(rot, theta, stretch="none", factor=1.0, original=8192, slow=1.0, fast=32.0):
    if stretch == "base":
        theta = theta * factor ** (rot / (rot - 2))
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if stretch == "linear":
        f = [x / factor for x in f]
    if stretch == "parts":
        g = [min(1.0, max(0.0, (original * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        f = [x * (a + (1 - a) / factor) for x, a in zip(f, g)]
    return f


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,dim,rot,layout,stretch", [
    (1, 1, 64, 64, "half", "none"), (7, 4, 256, 256, "half", "linear"), (33, 3, 128, 64, "interleaved", "parts"),
    (129, 5, 128, 32, "half", "base"), (5, 2, 80, 80, "interleaved", "none"), (3, 7, 96, 6, "half", "none"),
    (2, 3, 10, 2, "interleaved", "linear"), (4099, 32, 128, 128, "half", "parts"), (1, 2, 7, 4, "half", "none")])
def test_rope_rows(dtype, tokens, heads, dim, rot, layout, stretch):
    g = gen(tokens * 7 + dim)
    x = randn(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    factor = 1.0 if stretch == "none" else 8.0
    turns, mag = S.rope_turns(rot, 1e6, stretch, factor)
    f = freqs(rot, 1e6, stretch, factor)
    assert mag == pytest.approx(0.1 * math.log(8.0) + 1 if stretch == "parts" else 1.0)
    # one rounding of the result; cosine, sine, their factor and the two products in fp32 (8 units of fp32);
    # the angle to 2^-25 of a turn
    tol = (R.UNIT[dtype] + 8 * 2.0 ** -24 + 2 * math.pi * 2.0 ** -25) * mag * 2 * x.double().abs().amax()
    for inverse in (False, True):
        want = R.rotate(x, pos, f, layout, mag, inverse)
        out = torch.full_like(x, math.nan)
        S.rope_rows(out, x, pos, turns, layout=layout, magnitude=mag, inverse=inverse)
        assert (out.double() - want).abs().max() <= tol
        assert torch.equal(out[..., rot:], x[..., rot:])
    same = x.clone()
    S.rope_rows(same, same, pos, turns, layout=layout, magnitude=mag, inverse=True)
    assert torch.equal(same, out)


def test_rope_rows_strided_and_unaligned():
    """q inside fused rows, heads before tokens, and rows at odd element offsets."""
    g = gen(5)
    turns, _ = S.rope_turns(64, 1e4)
    f = freqs(64, 1e4)
    pos = torch.arange(50, 61, device="cuda", dtype=torch.int32)
    wide = randn(g, 11, 9, 64, dtype=F16)
    across = randn(g, 4, 11, 64, dtype=F16).transpose(0, 1)
    odd = randn(g, 11 * 4 * 64 + 3, dtype=F16)[3:].view(11, 4, 64)
    for x in (wide[:, 2:6], across, odd):
        out = torch.empty_like(x)
        before = x.clone()
        S.rope_rows(out, x, pos, turns)
        want = R.rotate(x, pos, f)
        assert (out.double() - want).abs().max() <= (2.0 ** -11 + 2.0 ** -20) * 2 * x.double().abs().amax()
        assert torch.equal(x, before)
    rest = wide.clone()
    S.rope_rows(wide[:, 2:6], wide[:, 2:6], pos, turns)
    assert torch.equal(wide[:, :2], rest[:, :2]) and torch.equal(wide[:, 6:], rest[:, 6:])


def test_rope_gradient():
    """The inverse with the forward's magnitude is its gradient: against the
    formula (the transpose of the rotation) and against central differences."""
    g = gen(9)
    turns, mag = S.rope_turns(64, 1e4, "parts", 4.0)
    pos = torch.randint(0, 9000, (6,), generator=g, device="cuda", dtype=torch.int32)
    x, w = randn(g, 6, 3, 64), randn(g, 6, 3, 64)

    def loss(y):
        out = torch.empty_like(y)
        S.rope_rows(out, y, pos, turns, magnitude=mag)
        return float((out.double() * w.double()).sum())

    grad = torch.empty_like(w)
    S.rope_rows(grad, w, pos, turns, magnitude=mag, inverse=True)
    want = R.rotate(w, pos, freqs(64, 1e4, "parts", 4.0), "half", mag, True)
    assert (grad.double() - want).abs().max() <= 2.0 ** -20 * mag * 2 * w.abs().amax()
    e = 2.0 ** -3  # the loss is linear in x: a large step costs nothing
    for t, h, d in ((0, 0, 0), (2, 1, 31), (3, 2, 32), (5, 0, 63)):
        up, down = x.clone(), x.clone()
        up[t, h, d] += e
        down[t, h, d] -= e
        assert (loss(up) - loss(down)) / (2 * e) == pytest.approx(float(grad[t, h, d]), abs=1e-4)


# ---- the cache ----------------------------------------------------------------
def make_cache(g, pages, page, heads, dim, dtype, garbage=True):
    k, v, ks, vs = S.new_pages(pages, page, heads, dim, dtype)
    if garbage:
        for t in (k, v):
            x = randn(g, *t.shape, std=TOPS.get(dtype, 4.0) / 4)
            x = x.clamp(-TOPS.get(dtype, 1e4), TOPS.get(dtype, 1e4))
            (t.view(torch.uint8) if dtype == FP8 else t).copy_(
                x.to(FP8).view(torch.uint8) if dtype == FP8 else x.round().to(I8) if dtype == I8 else x.to(dtype))
        for s in (ks, vs):
            if s is not None:
                s.uniform_(0.5, 1.5, generator=g).mul_(4 / TOPS[dtype])
    return k, v, ks, vs


TOPS = {I8: 127.0, FP8: 448.0}


@pytest.mark.parametrize("cache", [I8, FP8, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,heads,dim,page,rot,layout", [
    (1, 1, 64, 8, 0, "half"), (37, 3, 128, 16, 64, "half"), (130, 1, 256, 64, 256, "interleaved"),
    (65, 2, 64, 256, 32, "interleaved"), (300, 8, 128, 32, 128, "half")])
def test_kv_write_and_read(cache, dtype, tokens, heads, dim, page, rot, layout):
    g = gen(tokens + dim)
    pages = (2 * tokens) // page + 2
    kp, vp, ks, vs = make_cache(g, pages, page, heads, dim, cache)
    old = [None if t is None else t.clone() for t in (kp, vp, ks, vs)]
    k, v = randn(g, tokens, heads, dim, dtype=dtype, std=2.0), randn(g, tokens, heads, dim, dtype=dtype, std=0.1)
    if tokens > 2:
        v[1] = 0
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    live = torch.ones(tokens, dtype=torch.bool, device="cuda")
    if tokens > 20:  # padding, and slots past the cache
        slots[3], slots[17] = -1, pages * page
        live[3] = live[17] = False
    pos = torch.randint(0, 100000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    turns = S.rope_turns(rot, 1e6)[0] if rot else None
    S.kv_write(kp, vp, ks, vs, k, v, slots, positions=pos if rot else None, turns=turns, layout=layout)
    # every other row is as it was
    untouched = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    untouched[slots[live]] = False
    rest = untouched.nonzero().flatten()
    for a, b in zip((kp, vp), old[:2]):
        assert torch.equal(a.view(torch.uint8)[rest // page, :, rest % page], b.view(torch.uint8)[rest // page, :, rest % page])
    kx = R.rotate(k, pos, freqs(rot, 1e6), layout) if rot else k.double()
    for pages_, scale, x, exact in ((kp, ks, kx, not rot), (vp, vs, v.double(), True)):
        got = R.rows_of(pages_, scale, slots[live])
        x = x[live]
        if cache in TOPS:
            top = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
            unit = top / TOPS[cache]
            # half a step of int8, or 2^-4 of the value and half of the smallest step of e4m3, and fp32 arithmetic
            step = 0.5 * unit if cache == I8 else torch.maximum(x.abs() * 2.0 ** -4, unit * 2.0 ** -10)
            assert ((got - x).abs() <= step + 2.0 ** -18 * top).all()
            if exact and scale is not None:  # the documented arithmetic, bit for bit
                y = (k if pages_ is kp else v)[live].float()
                m = y.abs().amax(-1).clamp(min=2.0 ** -100)
                q = torch.full_like(m, TOPS[cache])
                code = y * (q / m)[..., None]
                code = code.round().clamp(-127, 127).to(I8) if cache == I8 else code.to(FP8)
                at = slots[live] // page, slice(None), slots[live] % page
                assert torch.equal(pages_.view(torch.uint8)[at], code.view(torch.uint8))
                assert torch.equal(scale[at], m / q)
        else:
            assert ((got - x).abs() <= (R.UNIT[cache] + 2.0 ** -18 * (not exact)) * x.abs().amax() + 2.0 ** -25).all()
    # reading: the same values, zeros for slots outside
    ko, vo = torch.full_like(k, math.nan), torch.full_like(v, math.nan)
    S.kv_read(kp, vp, ks, vs, ko, vo, slots)
    for out, pages_, scale in ((ko, kp, ks), (vo, vp, vs)):
        want = R.rows_of(pages_, scale, slots[live])
        assert ((out[live].double() - want).abs() <= (R.UNIT[dtype] + 2.0 ** -23) * want.abs() + 2.0 ** -25).all()
        assert not out[~live].any()


@pytest.mark.parametrize("cache", [I8, FP8])
def test_kv_rows_that_are_not_finite_or_tiny(cache):
    kp, vp, ks, vs = S.new_pages(2, 8, 1, 64, cache)
    k = torch.ones(6, 1, 64, device="cuda")
    v = torch.ones(6, 1, 64, device="cuda")
    k[0, 0, 5], k[1, 0, 0], v[2, 0, 63] = math.inf, math.nan, -math.inf
    k[3], k[4], v[5] = 0.0, 1e-38, 3e38
    slots = torch.arange(6, device="cuda")
    S.kv_write(kp, vp, ks, vs, k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    S.kv_read(kp, vp, ks, vs, ko, vo, slots)
    assert torch.isnan(ko[:2]).all() and torch.isnan(vo[2]).all()
    assert torch.isfinite(ko[2:]).all() and torch.isfinite(vo[[0, 1, 3, 4, 5]]).all()
    assert not ko[3].any() and ko[4].abs().max() < 1e-30
    assert ((vo[5] / 3e38) - 1).abs().max() < 2.0 ** -20


def test_kv_offsets_past_32_bits():
    """A cache whose last rows lie beyond element 2^32."""
    page, dim, heads = 256, 256, 8
    pages = (1 << 32) // (page * dim * heads) + 2
    kp, vp = (torch.empty(pages, heads, page, dim, dtype=I8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, heads, page, device="cuda") for _ in range(2))
    g = gen(3)
    k, v = randn(g, 3, heads, dim, dtype=F16), randn(g, 3, heads, dim, dtype=F16)
    slots = ints([pages * page - 1, (pages - 1) * page, 5], torch.int64)
    S.kv_write(kp, vp, ks, vs, k, v, slots)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    S.kv_read(kp, vp, ks, vs, ko, vo, slots)
    for x, y in ((k, ko), (v, vo)):
        assert ((x.float() - y.float()).abs() <= x.float().abs().amax(-1, keepdim=True) * (0.5 / 127 + 2.0 ** -11)).all()
    # and attention reads them
    q = randn(g, 1, heads, dim, dtype=F16)
    sc = S.new_scratch()
    out = torch.empty_like(q)
    S.attention_paged(out, q, kp, vp, ks, vs, ints([[pages - 1]]), ints([1]), ints([0, 1]), 1, sc)
    want = R.rows_of(vp, vs, slots[1:2])
    assert ((out.double() - want).abs() <= 2.0 ** -10 * want.abs() + 1e-6).all()


# ---- attention ------------------------------------------------------------------
def check_attention(out, lse, want, mag, wlse, dtype, keys, vmax):
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(out)), "finite where it should not be, or the other way round"
    off = (out.double() - want).abs() - R.attention_bound(want, mag, dtype, keys, vmax)
    assert off[fine].max() <= 0, float(off[fine].max())
    if lse is not None:
        none = wlse == -math.inf
        assert torch.equal(lse == -math.inf, none)
        # scores to 2^-12 (fp32 dot products of up to 256 terms), and fp32 of the result
        assert ((lse.double() - wlse).abs()[~none] <= 2.0 ** -12 + 2.0 ** -22 * wlse.abs()[~none]).all()


def run_packed(scratch, lens, heads, kv_heads, dim, dtype, window=0, scale=0.0, seed=0, fused=False, edit=None,
               extra=0):
    g = gen(seed)
    n = sum(lens) + extra
    if fused:
        x = randn(g, n, heads + 2 * kv_heads, dim, dtype=dtype)
        q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    else:
        q, k, v = (randn(g, n, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    if edit:
        edit(q, k, v)
    out = torch.full((n, heads, dim), math.nan, dtype=dtype, device="cuda")
    lse = torch.full((n, heads), math.nan, device="cuda")
    S.attention_packed(out, q, k, v, starts_of(lens), scratch, window=window, scale=scale, lse=lse)
    assert S.error_word(scratch) == 0
    at = 0
    for m in lens:
        s = slice(at, at + m)
        want, mag, wlse = R.attend(q[s], k[s], v[s], 0, window, scale or dim ** -0.5)
        vmax = float(torch.nan_to_num(v[s].float(), posinf=0, neginf=0).abs().max()) if m else 0.0
        if m:
            check_attention(out[s], lse[s], want, mag, wlse, dtype, m, vmax)
        at += m
    assert not out[at:].any() and (lse[at:] == -math.inf).all()
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,heads,kv_heads,window", [
    ([1], 1, 1, 0), ([1, 0, 2, 0], 4, 1, 0), ([127, 128, 129], 4, 4, 0), ([5, 300, 1, 64], 6, 2, 0),
    ([513], 7, 1, 0), ([260, 31], 4, 1, 1), ([700, 3], 4, 2, 100), ([1025], 3, 3, 512), ([33, 200], 8, 1, 4096)])
def test_packed(scratch, dtype, dim, lens, heads, kv_heads, window):
    run_packed(scratch, lens, heads, kv_heads, dim, dtype, window, seed=sum(lens) + dim)


def test_packed_long_and_fused(scratch):
    run_packed(scratch, [2500, 1, 777], 8, 2, 128, BF16, fused=True, seed=1)
    run_packed(scratch, [3001], 4, 1, 256, F16, fused=True, window=512, scale=0.2, seed=2)
    run_packed(scratch, [1500, 1501], 2, 2, 64, F16, fused=True, seed=3)


def test_packed_tokens_in_no_sequence(scratch):
    run_packed(scratch, [70, 5], 4, 1, 128, F16, extra=9, seed=4)


def test_packed_many_short(scratch):
    r = random.Random(4)
    run_packed(scratch, [r.choice([0, 1, 1, 2, 3, 17]) for _ in range(150)], 4, 2, 64, BF16, seed=6)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_packed_large_scores(scratch, dim):
    """Scores of hundreds, all negative for some rows: the running maximum has
    to hold, and the weights of far keys vanish."""
    def edit(q, k, v):
        q.mul_(8)
        k[100:].mul_(6)
        k[40:80].copy_(-q[40:80, :1] * 2)
    g = gen(0)
    x = [randn(g, 400, h, dim, dtype=F16) for h in (2, 1, 1)]
    edit(*x)
    out, lse = torch.empty_like(x[0]), torch.empty(400, 2, device="cuda")
    S.attention_packed(out, *x, ints([0, 400]), scratch, lse=lse)
    want, mag, wlse = R.attend(*x, 0, 0, dim ** -0.5)
    # scores in the hundreds: their fp32 error is 2^-13 of the bound's for scores near 10, scaled up
    top = float(wlse.abs().max())
    tol = R.attention_bound(want, mag, F16, 400, float(x[2].abs().max())) + mag * top * 2.0 ** -17
    assert ((out.double() - want).abs() <= tol).all()
    assert ((lse.double() - wlse).abs() <= top * 2.0 ** -17).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_packed_what_is_masked_does_not_matter(scratch, dim, window, bad):
    """An infinity or NaN in k or v of one token reaches exactly the tokens that attend to it."""
    def edit(q, k, v):
        v[150, 0, 3] = bad
        v[399, 0, dim - 1] = bad
        k[300, 0, 7] = bad
        v[530, 0, 0] = bad
    g = gen(dim)
    lens = [400, 140]
    q, k, v = (randn(g, 540, h, dim, dtype=BF16) for h in (4, 1, 1))
    edit(q, k, v)
    out = torch.zeros_like(q)
    S.attention_packed(out, q, k, v, starts_of(lens), scratch, window=window)
    at = 0
    for m in lens:
        s = slice(at, at + m)
        want, mag, _ = R.attend(q[s], k[s], v[s], 0, window, dim ** -0.5)
        # a row that sees a NaN key, or an infinite one on its side, is NaN altogether; the others stay as they are
        fine = torch.isfinite(want)
        assert torch.equal(torch.isfinite(out[s]), fine)
        tol = R.attention_bound(want, mag, BF16, m, 6.0)
        assert ((out[s].double() - want).abs() <= tol)[fine].all()
        at += m


def run_paged(scratch, q_lens, kv_lens, heads, kv_heads, dim, page, cache, dtype, window=0, seed=0, poison=True,
              scale=0.0, width=0):
    g = gen(seed)
    held = [-(-n // page) for n in kv_lens]
    pages = sum(held) + 3
    kp, vp, ks, vs = make_cache(g, pages, page, kv_heads, dim, cache)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = width or max(max(held), 1) + 1
    table, at = torch.full((len(kv_lens), width), -1, dtype=torch.int32), 0
    slots = []
    for b, n in enumerate(held):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        i = torch.arange(kv_lens[b])
        slots.append((table[b, i // page].long() * page + i % page).cuda())
        at += n
    if poison:  # every row that no sequence holds: NaN
        free = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        for s in slots:
            free[s] = False
        free = free.nonzero().flatten()
        for p, s in ((kp, ks), (vp, vs)):
            if s is None:
                p[free // page, :, free % page] = math.nan
            else:
                s[free // page, :, free % page] = math.nan
                p.view(torch.uint8)[free // page, :, free % page] = 0x7F
    n = sum(q_lens)
    q = randn(g, n, heads, dim, dtype=dtype)
    out = torch.full((n, heads, dim), math.nan, dtype=dtype, device="cuda")
    lse = torch.full((n, heads), math.nan, device="cuda")
    S.attention_paged(out, q, kp, vp, ks, vs, table.cuda(), ints(kv_lens), starts_of(q_lens), max(q_lens + [1]),
                      scratch, window=window, scale=scale, lse=lse)
    assert S.error_word(scratch) == 0
    at = 0
    for b, m in enumerate(q_lens):
        s = slice(at, at + m)
        k, v = R.rows_of(kp, ks, slots[b]), R.rows_of(vp, vs, slots[b])
        want, mag, wlse = R.attend(q[s], k, v, kv_lens[b] - m, window, scale or dim ** -0.5)
        if m:
            check_attention(out[s], lse[s], want, mag, wlse, dtype, max(kv_lens[b], 1),
                            float(v.abs().max()) if kv_lens[b] else 0.0)
        at += m


CACHES = [(F16, F16), (BF16, BF16), (I8, F16), (I8, BF16), (FP8, F16), (FP8, BF16)]


@pytest.mark.parametrize("cache,dtype", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads,page,window", [
    ([1], [1], 1, 1, 16, 0), ([1, 1, 0, 1], [130, 1, 0, 2000], 4, 1, 16, 0), ([1] * 5, [64, 65, 127, 128, 129], 8, 8, 8, 0),
    ([1, 3, 4, 2], [700, 300, 4, 5], 8, 2, 32, 0), ([1, 1], [3000, 40], 5, 1, 64, 512), ([2, 1], [600, 90], 16, 1, 128, 1),
    ([1], [1500], 64, 2, 256, 0)])
def test_paged_few_rows(scratch, cache, dtype, dim, q_lens, kv_lens, heads, kv_heads, page, window):
    run_paged(scratch, q_lens, kv_lens, heads, kv_heads, dim, page, cache, dtype, window, seed=dim + sum(kv_lens))


@pytest.mark.parametrize("cache,dtype", CACHES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,kv_lens,heads,kv_heads,page,window", [
    ([40], [40], 4, 1, 16, 0), ([17, 0, 130, 1], [500, 0, 131, 900], 4, 2, 8, 0), ([300], [1111], 6, 1, 64, 0),
    ([64, 200], [2000, 200], 4, 1, 16, 300), ([129], [129], 3, 3, 128, 7)])
def test_paged_chunks(scratch, cache, dtype, dim, q_lens, kv_lens, heads, kv_heads, page, window):
    run_paged(scratch, q_lens, kv_lens, heads, kv_heads, dim, page, cache, dtype, window, seed=dim + sum(kv_lens))


@pytest.mark.parametrize("q_lens,kv_lens", [([3, 2], [0, 1]), ([50, 200], [20, 0]), ([1], [0])])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_paged_rows_that_see_nothing(scratch, q_lens, kv_lens, dim):
    """More new tokens than keys: the first sit at negative positions."""
    run_paged(scratch, q_lens, kv_lens, 4, 1, dim, 16, I8, F16)
    run_paged(scratch, q_lens, kv_lens, 4, 2, dim, 16, BF16, BF16)


def test_paged_long_context(scratch):
    run_paged(scratch, [1], [40001], 4, 1, 256, 16, F16, F16, seed=1)
    run_paged(scratch, [1, 1, 1], [20000, 7, 30000], 8, 2, 128, 64, FP8, BF16, seed=2)
    run_paged(scratch, [20], [20000], 4, 1, 256, 64, I8, BF16, seed=3)
    run_paged(scratch, [33, 1], [17000, 9000], 16, 2, 128, 32, BF16, BF16, seed=4)
    run_paged(scratch, [5], [33000], 2, 1, 64, 128, I8, F16, seed=5)


def test_paged_many_sequences(scratch):
    r = random.Random(1)
    kv = [r.choice([0, 1, 5, 130, 700, 2049]) for _ in range(200)]
    run_paged(scratch, [min(1, n) for n in kv], kv, 4, 2, 64, 16, FP8, F16, seed=7)
    q = [min(n, r.choice([0, 1, 2, 30])) for n in kv]
    run_paged(scratch, q, kv, 4, 2, 64, 16, I8, BF16, seed=8)


@pytest.mark.parametrize("q_len", [1, 40])
def test_paged_window_never_reads_pages_left_behind(scratch, q_len):
    """Pages before every window may be gone from the table."""
    g = gen(11)
    kv, window, page = 1000, 100, 16
    kp, vp, ks, vs = make_cache(g, 70, page, 1, 128, I8)
    table = torch.arange(63, dtype=torch.int32, device="cuda")[None].contiguous()
    q = randn(g, q_len, 4, 128, dtype=F16)
    outs = []
    for gone in (False, True):
        if gone:
            table[0, : (kv - q_len - window + 1) // page] = -1
        out = torch.empty_like(q)
        S.attention_paged(out, q, kp, vp, ks, vs, table, ints([kv]), ints([0, q_len]), q_len, scratch, window=window)
        assert S.error_word(scratch) == 0
        outs.append(out)
    assert torch.equal(*outs)


def test_paged_zero_values_and_uneven_scales(scratch):
    """Rows of zeros, and rows whose scales differ by 2^40: each key weighs by its score alone."""
    g = gen(21)
    for cache in (I8, FP8):
        for n in (1, 30):
            for dim in (64, 256):
                kp, vp, ks, vs = S.new_pages(20, 16, 1, dim, cache)
                k, v = randn(g, 300, 1, dim), randn(g, 300, 1, dim)
                v[7:90] = 0
                v[120:140] *= 2.0 ** -40
                slots = torch.arange(300, device="cuda")
                S.kv_write(kp, vp, ks, vs, k, v, slots)
                q = randn(g, n, 4, dim, dtype=BF16, std=2.0)
                out, lse = torch.empty_like(q), torch.empty(n, 4, device="cuda")
                S.attention_paged(out, q, kp, vp, ks, vs, torch.arange(20, dtype=torch.int32, device="cuda")[None],
                                  ints([300]), ints([0, n]), n, scratch, lse=lse)
                want, mag, wlse = R.attend(q, R.rows_of(kp, ks, slots), R.rows_of(vp, vs, slots), 300 - n, 0, dim ** -0.5)
                check_attention(out, lse, want, mag, wlse, BF16, 300, 5.0)
                # nothing but zeros
                vp.view(torch.uint8).zero_()
                S.attention_paged(out, q, kp, vp, ks, vs, torch.arange(20, dtype=torch.int32, device="cuda")[None],
                                  ints([300]), ints([0, n]), n, scratch)
                assert not out.any()


@pytest.mark.parametrize("n", [1, 60])
def test_paged_bad_tables_and_lengths_are_reported(scratch, n):
    g = gen(13)
    kp, vp, ks, vs = make_cache(g, 8, 16, 1, 64, F16)
    q = randn(g, n, 2, 64, dtype=F16)
    out = torch.empty_like(q)
    S.attention_paged(out, q, kp, vp, ks, vs, ints([[0, 8, 2, 3, 4]]), ints([80]), ints([0, n]), n, scratch)
    assert S.error_word(scratch) == 2
    zero = [t.clone() for t in (kp, vp)]
    for t in zero:
        t[1] = 0
    want = torch.empty_like(q)
    S.attention_paged(want, q, *zero, ks, vs, ints([[0, 1, 2, 3, 4]]), ints([80]), ints([0, n]), n, scratch)
    assert torch.equal(out, want)
    S.attention_paged(out, q, kp, vp, ks, vs, ints([[0, 1, 2, 3, 4]]), ints([900]), ints([0, n]), n, scratch)
    assert S.error_word(scratch) == 1
    S.attention_paged(out, q, kp, vp, ks, vs, ints([[0, 1, 2, 3, 4]]), ints([80]), ints([0, n]), n, scratch)
    assert S.error_word(scratch) == 0
    if n > 1:
        S.attention_paged(out, q, kp, vp, ks, vs, ints([[0, 1, 2, 3, 4]]), ints([80]), ints([0, n]), 1, scratch)
        assert S.error_word(scratch) == 8


def test_starts_that_make_no_sense_stay_inside(scratch):
    g = gen(14)
    x = [randn(g, 64, h, 128, dtype=F16) for h in (4, 1, 1)]
    out = torch.empty_like(x[0])
    S.attention_packed(out, *x, ints([-5, 40, 20, 9000]), scratch)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_results_do_not_vary_and_streams_are_kept(scratch, dim):
    """The same call twice gives the same bits, alone, after other work in the same scratch, and on another stream."""
    g = gen(15)
    x = [randn(g, 900, h, dim, dtype=BF16) for h in (8, 2, 2)]
    kp, vp, ks, vs = make_cache(g, 600, 16, 2, dim, FP8)
    table = torch.randperm(600, generator=g, device="cuda", dtype=torch.int32)[None].contiguous()
    stream = torch.cuda.Stream()

    def both():
        a, b, c = torch.empty_like(x[0]), torch.empty_like(x[0][:1]), torch.empty_like(x[0][:50])
        S.attention_packed(a, *x, ints([0, 200, 900]), scratch)
        S.attention_paged(b, x[0][:1], kp, vp, ks, vs, table, ints([9600]), ints([0, 1]), 1, scratch)
        S.attention_paged(c, x[0][:50], kp, vp, ks, vs, table, ints([9600]), ints([0, 50]), 50, scratch)
        return a, b, c

    first = both()
    second = both()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        third = both()
    stream.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_calls_can_be_captured(scratch):
    """All operators in one CUDA graph, replayed on new inputs."""
    g = gen(17)
    kp, vp, ks, vs = make_cache(g, 64, 16, 1, 256, I8)
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None].contiguous()
    turns, _ = S.rope_turns(256, 1e6)
    q, k, v = (randn(g, 1, h, 256, dtype=F16) for h in (4, 1, 1))
    qr, out = torch.empty_like(q), torch.empty_like(q)
    pos, lens, slots = ints([1000]), ints([1001]), ints([1000], torch.int64)
    one = ints([0, 1])

    def step():
        S.rope_rows(qr, q, pos, turns)
        S.kv_write(kp, vp, ks, vs, k, v, slots, positions=pos, turns=turns)
        S.attention_paged(out, qr, kp, vp, ks, vs, table, lens, one, 1, scratch)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        q.copy_(randn(g, 1, 4, 256, dtype=F16))
        k.copy_(randn(g, 1, 1, 256, dtype=F16))
        pos.add_(1)
        lens.add_(1)
        slots.add_(1)
        graph.replay()
        replayed = out.clone()
        step()
        assert torch.equal(replayed, out)


def test_no_tokens_is_no_work(scratch):
    x = [torch.empty(0, h, 128, dtype=F16, device="cuda") for h in (4, 1, 1)]
    S.attention_packed(x[0], *x, ints([0, 0]), scratch)
    S.rope_rows(x[0], x[0], ints([]), S.rope_turns(128, 1e4)[0])
    kp, vp, ks, vs = S.new_pages(4, 16, 1, 128, I8)
    S.kv_write(kp, vp, ks, vs, x[1], x[2], ints([], torch.int64))
    S.kv_read(kp, vp, ks, vs, x[1], x[2], ints([], torch.int64))
    S.attention_paged(x[0], x[0], kp, vp, ks, vs, ints([[0], [0]]), ints([3, 0]), ints([0, 0, 0]), 1, scratch)
    torch.cuda.synchronize()


# ---- layouts, and what only some kernels meet ------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_packed_layouts_and_shared_heads(scratch, dim):
    """Heads before tokens, one k and v head broadcast to several, and rows far apart."""
    g = gen(31)
    n, lens = 333, [200, 133]
    q = randn(g, 6, n, dim, dtype=BF16).transpose(0, 1)
    k, v = (randn(g, n, 1, dim, dtype=BF16).expand(n, 3, dim) for _ in range(2))
    assert k.stride(1) == 0
    far = torch.zeros(n, 9, dim, dtype=BF16, device="cuda")
    out, lse = far[:, 2:8], torch.empty(n, 6, device="cuda")
    S.attention_packed(out, q, k, v, starts_of(lens), scratch, lse=lse)
    at = 0
    for m in lens:
        s = slice(at, at + m)
        want, mag, wlse = R.attend(q[s], k[s], v[s], 0, 0, dim ** -0.5)
        check_attention(out[s], lse[s], want, mag, wlse, BF16, m, 5.0)
        at += m
    assert not far[:, :2].any() and not far[:, 8:].any()


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 128, 1), (3, 100, 2), (40, 64, 1), (200, 33, 33)])
def test_paged_unusual_groups(scratch, rows, heads, kv_heads):
    run_paged(scratch, [rows, 1], [rows + 300, 77], heads, kv_heads, 64, 16, I8, BF16, seed=rows)
    run_paged(scratch, [rows], [rows + 140], heads, kv_heads, 128, 32, F16, F16, window=50, seed=rows + 1)


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 3e4, 1e30])
@pytest.mark.parametrize("n", [1, 50])
def test_paged_queries_of_any_size(scratch, cache, size, n):
    """bf16 queries far outside fp16's range over 8-bit pages: the scale of the scores makes up for it."""
    g = gen(33)
    kp, vp, ks, vs = make_cache(g, 40, 16, 1, 256, cache)
    table = torch.randperm(40, generator=g, device="cuda", dtype=torch.int32)[None].contiguous()
    q = (torch.randn(n, 4, 256, generator=g, device="cuda") * size).to(BF16)
    q[0, 1] = 0
    out, lse = torch.empty_like(q), torch.empty(n, 4, device="cuda")
    scale = 0.0625 / size
    S.attention_paged(out, q, kp, vp, ks, vs, table, ints([600]), ints([0, n]), n, scratch, scale=scale, lse=lse)
    i = torch.arange(600, device="cuda")
    slots = table[0, i // 16].long() * 16 + i % 16
    want, mag, wlse = R.attend(q, R.rows_of(kp, ks, slots), R.rows_of(vp, vs, slots), 600 - n, 0,
                               float(torch.tensor(scale, dtype=F32)))
    check_attention(out, lse, want, mag, wlse, BF16, 600, float(vs.max()) * TOPS[cache])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,window", [(4, 0), (4, 100), (60, 0), (60, 100), (1, 100)])
def test_paged_what_is_masked_does_not_matter(scratch, dtype, dim, n, window):
    """Infinities and NaN in 16-bit pages reach exactly the new tokens that see them."""
    g = gen(35)
    kv, page = 700, 16
    kp, vp, ks, vs = make_cache(g, 44, page, 1, dim, dtype)
    table = torch.arange(44, dtype=torch.int32, device="cuda")[None].contiguous()
    at = lambda j: (j // page, 0, j % page)  # noqa: E731
    vp[at(698)][3], vp[at(699)][dim - 1] = math.nan, math.inf
    kp[at(697)][1] = math.nan
    vp[at(kv - n - window + 2 if window else 5)][0] = -math.inf
    q = randn(g, n, 2, dim, dtype=dtype)
    out = torch.empty_like(q)
    S.attention_paged(out, q, kp, vp, ks, vs, table, ints([kv]), ints([0, n]), n, scratch, window=window)
    slots = torch.arange(kv, device="cuda")
    want, mag, _ = R.attend(q, R.rows_of(kp, ks, slots), R.rows_of(vp, vs, slots), kv - n, window, dim ** -0.5)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine)
    assert ((out.double() - want).abs() <= R.attention_bound(want, mag, dtype, kv, 6.0))[fine].all()


@pytest.mark.parametrize("n", [1, 4, 30])
def test_paged_rows_written_as_nan(scratch, n):
    """A token whose values were not finite makes those who see it NaN, and nobody else."""
    g = gen(37)
    kp, vp, ks, vs = S.new_pages(20, 16, 1, 64, I8)
    k, v = randn(g, 300, 1, 64), randn(g, 300, 1, 64)
    v[290, 0, 9] = math.inf
    S.kv_write(kp, vp, ks, vs, k, v, torch.arange(300, device="cuda"))
    q = randn(g, n, 2, 64, dtype=F16)
    out = torch.empty_like(q)
    for length in (290, 292, 300):
        S.attention_paged(out, q, kp, vp, ks, vs, torch.arange(20, dtype=torch.int32, device="cuda")[None].contiguous(),
                          ints([length]), ints([0, n]), n, scratch)
        sees = torch.arange(length - n, length, device="cuda") >= 290
        assert torch.equal(torch.isnan(out).all(-1).all(-1), sees) and torch.isfinite(out[~sees]).all()


def test_many_sequences_at_once(scratch):
    r = random.Random(9)
    kv = [r.choice([0, 1, 3, 20, 150]) for _ in range(1200)]
    run_paged(scratch, [min(1, n) for n in kv], kv, 2, 1, 64, 8, F16, F16, seed=10)
    run_paged(scratch, [min(n, r.choice([1, 9, 20])) for n in kv], kv, 2, 1, 64, 8, F16, F16, seed=11)


def test_python_refusals():
    x = torch.zeros(4, 2, 64, dtype=F16)
    c = x.cuda()
    kp, vp, ks, vs = S.new_pages(4, 16, 2, 64, I8)
    turns, _ = S.rope_turns(64, 1e4)
    pos, slots = ints([0, 1, 2, 3]), ints([0, 1, 2, 3], torch.int64)
    bad = [lambda: S.rope_rows(x, x, pos, turns), lambda: S.rope_rows(c, c, pos.long(), turns),
           lambda: S.rope_rows(c, c, pos[:3], turns), lambda: S.rope_rows(c, c, pos, turns, layout="other"),
           lambda: S.rope_rows(c[:, :, ::2], c[:, :, ::2], pos, turns), lambda: S.rope_rows(c[0], c[0], pos, turns),
           lambda: S.rope_rows(c.double(), c.double(), pos, turns), lambda: S.rope_rows(None, c, pos, turns),
           lambda: S.kv_write(kp, vp, None, None, c, c, slots), lambda: S.kv_write(kp, vp[:2], ks, vs, c, c, slots),
           lambda: S.kv_write(kp, vp, ks, vs, c, c, pos), lambda: S.kv_read(kp, vp, ks[:2], vs, c, c, slots),
           lambda: S.kv_write(kp, vp, ks, vs, c, c, slots, positions=None, turns=turns),
           lambda: S.attention_packed(c, c, c, c, ints([0, 4]), torch.zeros(100, dtype=torch.uint8, device="cuda")),
           lambda: S.attention_paged(c, c, kp, vp, ks, vs, ints([0, 1]), ints([4]), ints([0, 4]), 4, S.new_scratch()),
           lambda: S.attention_paged(c, c, kp, vp, ks, vs, ints([[0, 1]]), ints([4]), ints([0, 2, 4]), 4, S.new_scratch()),
           lambda: S.attention_paged(c, c, kp, vp, ks, vs, ints([[0, 1]]), ints([4]), ints([0, 4]), -1, S.new_scratch())]
    for f in bad:
        with pytest.raises(S.XpError):
            f()
