"""The serving operators at their edges: scales, codes, queries and devices that
ordinary use seldom meets, against the plain 64-bit forms."""
import random

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import serving_ref as R  # noqa: E402
from test_gpu_serving import check_attention, gen, ints, make_cache, randn  # noqa: E402
from xpose_b200 import serving as S  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
I8, FP8 = torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def scratch():
    return S.new_scratch()


def test_tensors_of_a_device_that_is_not_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    outs = []
    for device in ("cuda:0", "cuda:1"):
        torch.cuda.set_device(0)
        g = torch.Generator().manual_seed(3)
        q, k, v = (torch.randn(70, h, 64, generator=g).to(F16).to(device) for h in (4, 1, 1))
        pos = torch.arange(70, dtype=torch.int32, device=device)
        slots = torch.arange(70, device=device)
        turns, _ = S.rope_turns(64, 1e4, device=device)
        pages = S.new_pages(8, 16, 1, 64, I8, device=device)
        scratch = S.new_scratch(device)
        one = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
        S.rope_rows(q, q, pos, turns)
        S.kv_write(*pages, k, v, slots, positions=pos, turns=turns)
        a, b = torch.empty_like(q), torch.empty_like(q)
        S.attention_packed(a, q, k, v, one(0, 70), scratch)
        S.attention_paged(b, q, *pages, one(0, 1, 2, 3, 4)[None].contiguous(), one(70), one(0, 70), 70, scratch)
        assert S.error_word(scratch) == 0 and torch.cuda.current_device() == 0
        outs.append((a.cpu(), b.cpu()))
    for x, y in zip(*outs):
        assert torch.equal(x, y)

def paged(scratch, cache, q, kv, scale=0.0, window=0, page=16):
    """attention_paged of q's tokens, the newest of kv keys in `cache`, against the 64-bit form."""
    kp, vp, ks, vs = cache
    n, dim = q.shape[0], q.shape[2]
    table = torch.arange(-(-kv // page), dtype=torch.int32, device="cuda")[None].contiguous()
    out, lse = torch.full_like(q, float("nan")), torch.empty(n, q.shape[1], device="cuda")
    S.attention_paged(out, q, kp, vp, ks, vs, table, ints([kv]), ints([0, n]), n, scratch, scale=scale, window=window,
                      lse=lse)
    assert S.error_word(scratch) == 0
    slots = torch.arange(kv, device="cuda")
    k, v = R.rows_of(kp, ks, slots), R.rows_of(vp, vs, slots)
    return out, lse, R.attend(q, k, v, kv - n, window, scale or dim ** -0.5), v


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,window", [(1, 0), (4, 0), (8, 50), (30, 0), (70, 100)])
def test_paged_value_scales_of_zero_and_next_to_it(scratch, cache, dtype, dim, n, window):
    """A value is code * scale whatever the code: rows whose scale is zero or has
    no finite inverse are rows of (next to) nothing, which weigh as any other."""
    g = gen(dim + n)
    kv = 300
    pages = make_cache(g, 20, 16, 1, dim, cache)
    vs, ks = pages[3].view(-1), pages[2].view(-1)
    vs[7:40] = 0.0                     # some of a tile, some of a step
    vs[48:64], vs[64:70] = 2.0 ** -130, 2.0 ** -149
    vs[70:74], vs[74:78] = 2.0 ** -126, 2.0 ** -107
    vs[128:256] = 0.0                  # a whole tile
    vs[kv - 1] = vs[kv - n // 2] = 0.0  # only some rows see it
    ks[100:105] = 0.0
    q = randn(g, n, 2, dim, dtype=dtype)
    out, lse, (want, mag, wlse), v = paged(scratch, pages, q, kv, window=window)
    check_attention(out, lse, want, mag, wlse, dtype, kv, float(v.abs().max()))
    vs[:] = 0.0
    out, lse, (_, _, wlse), _ = paged(scratch, pages, q, kv, window=window)
    assert not out.any() and ((lse.double() - wlse).abs() <= 2.0 ** -12 + 2.0 ** -22 * wlse.abs()).all()


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("n", [1, 30])
def test_paged_rows_of_zeros_keep_their_weight_beside_large_values(scratch, cache, n):
    """Two thousand keys without values, each e^-12 of one key with values near 3e4, take 1.2 % of its weight."""
    kv, dim = 2048, 64
    pages = S.new_pages(kv // 16, 16, 1, dim, cache)
    k, v = torch.zeros(kv, 1, dim, device="cuda"), torch.zeros(kv, 1, dim, device="cuda")
    k[5, 0, 0] = 12.0
    v[5] = 3e4
    S.kv_write(*pages, k, v, torch.arange(kv, device="cuda"))
    q = torch.zeros(n, 1, dim, dtype=BF16, device="cuda")
    q[:, 0, 0] = 1.0
    out, lse, (want, mag, wlse), v = paged(scratch, pages, q, kv, scale=1.0)
    assert float(want[-1].max()) < 0.99 * 3e4
    check_attention(out, lse, want, mag, wlse, BF16, 0, 0.0)


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("n", [1, 30])
def test_paged_codes_of_nan_under_a_scale_of_zero_are_zeros(scratch, cache, n):
    """A row that was never written holds any codes."""
    g = gen(39)
    kv, dim = 300, 128
    pages = make_cache(g, 20, 16, 1, dim, cache)
    pages[3].view(-1)[40:60] = 0.0
    clean = paged(scratch, pages, q := randn(g, n, 2, dim, dtype=BF16), kv)[0]
    pages[1].view(torch.uint8).view(-1, dim)[40:60] = 0x7F
    assert torch.isfinite(clean).all()
    table = torch.arange(19, dtype=torch.int32, device="cuda")[None].contiguous()
    out = torch.empty_like(q)
    S.attention_paged(out, q, *pages, table, ints([kv]), ints([0, n]), n, scratch)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("scale", [2.0 ** -106, 2.0 ** 120, 2.0 ** 126, 2.0 ** 127])
@pytest.mark.parametrize("n", [1, 30])
def test_paged_value_scales_of_any_size(scratch, cache, scale, n):
    """... and those whose inverse is subnormal, or whose values are near the ends of fp32."""
    g = gen(40)
    kv, dim = 300, 64
    pages = make_cache(g, 20, 16, 1, dim, cache)
    v = torch.randint(-1, 2, pages[1].shape, generator=g, device="cuda").float()
    pages[1].view(torch.uint8).copy_(v.to(cache).view(torch.uint8))
    pages[3].fill_(scale)
    out, lse, (want, mag, wlse), v = paged(scratch, pages, randn(g, n, 2, dim, dtype=BF16), kv)
    check_attention(out, lse, want, mag, wlse, BF16, kv, scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,window", [(4, 0), (4, 100), (8, 0), (60, 0), (60, 100), (200, 0), (1, 100)])
def test_paged_codes_that_are_nan_reach_those_who_see_them(scratch, dtype, dim, n, window):
    """e4m3 has codes of NaN. With an ordinary scale beside them they are NaN in
    their own place, for the new tokens that see the key and for nobody else."""
    g = gen(41 + dim)
    kv, page = 700, 16
    pages = make_cache(g, 44, page, 1, dim, FP8)
    kb, vb = (t.view(torch.uint8).view(44, page, dim) for t in pages[:2])
    at = lambda j: (j // page, j % page)  # noqa: E731
    vb[at(698)][3], vb[at(699)][dim - 1] = 0x7F, 0xFF
    vb[at(kv - n + 1)][17] = 0x7F
    kb[at(697)][1] = 0xFF
    vb[at(kv - n - window + 2 if window else 5)][0] = 0x7F
    q = randn(g, n, 2, dim, dtype=dtype)
    out, _, (want, mag, _), v = paged(scratch, pages, q, kv, window=window)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine)
    assert fine.any() or n == 1 or not window  # a token before the NaN keys is left as it is
    top = float(torch.nan_to_num(v).abs().max())
    assert ((out.double() - want).abs() <= R.attention_bound(want, mag, dtype, kv, top))[fine].all()


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("exponent", [122, 123, 126, 127])
@pytest.mark.parametrize("n", [1, 40])
def test_paged_largest_finite_queries(scratch, cache, exponent, n):
    """bf16 queries up to the type's largest, over keys of -1, 0 and 1 in the
    places where they are: the dot products stay within fp32."""
    g = gen(43)
    kv, dim = 300, 64
    pages = make_cache(g, 20, 16, 1, dim, cache)
    k = torch.randint(-1, 2, (20, 1, 16, dim), generator=g, device="cuda").float()
    k[..., 1:] = 0
    pages[0].view(torch.uint8).copy_(k.to(cache).view(torch.uint8))
    pages[2].fill_(1.0)
    q = torch.zeros(n, 2, dim, device="cuda")
    q[..., 0] = (torch.rand(n, 2, generator=g, device="cuda") * 0.9 + 1.0) * 2.0 ** 60
    q = (q * 2.0 ** (exponent - 60)).to(BF16)
    assert torch.isfinite(q).all()
    out, lse, (want, mag, wlse), v = paged(scratch, pages, q, kv, scale=2.0 ** -(exponent - 1))
    check_attention(out, lse, want, mag, wlse, BF16, kv, float(v.abs().max()))


@pytest.mark.parametrize("pages", [True, False])
def test_256_wide_tiles_one_after_the_other_never_lose_a_wait(pages):
    """Thousands of calls in a row, whose row tiles end at all moments: no wait
    runs out, whichever warp comes late to the last products of its tile."""
    g = gen(51)
    new, kv = [512, 37, 60, 101, 331], [8192, 600, 1000, 2300, 5000]
    scratch, starts, n = S.new_scratch(), [0], sum(new)
    for m in new:
        starts.append(starts[-1] + m)
    q = randn(g, n, 4, 256, dtype=BF16)
    out = torch.empty_like(q)
    if pages:
        held = [-(-m // 16) for m in kv]
        cache = make_cache(g, sum(held), 16, 1, 256, I8)
        table = torch.full((len(kv), max(held)), -1, dtype=torch.int32)
        order = torch.randperm(sum(held), generator=g, device="cuda", dtype=torch.int32).cpu()
        for b, m in enumerate(held):
            table[b, :m] = order[sum(held[:b]):sum(held[:b]) + m]
        table, lens = table.cuda(), ints(kv)
        call = lambda: S.attention_paged(out, q, *cache, table, lens, ints_starts, 512, scratch)  # noqa: E731
    else:
        k, v = randn(g, n, 1, 256, dtype=BF16), randn(g, n, 1, 256, dtype=BF16)
        call = lambda: S.attention_packed(out, q, k, v, ints_starts, scratch, window=300)  # noqa: E731
    ints_starts = ints(starts)
    call()
    first = out.clone()
    for _ in range(10):
        for _ in range(1000):
            call()
        assert S.error_word(scratch) == 0
        assert torch.equal(out, first)


@pytest.mark.parametrize("cache", [I8, FP8])
@pytest.mark.parametrize("exponent", [-40, -4, -3, -1, 0, 3, 14, 15])
@pytest.mark.parametrize("n", [1, 50])
def test_paged_queries_of_mixed_sizes(scratch, cache, exponent, n):
    """bf16 queries whose scores come from values 2^-16 of the row's largest,
    which meets keys of zero there: they enter whole, wherever the largest is."""
    g = gen(47)
    kv, dim = 300, 64
    pages = make_cache(g, 20, 16, 1, dim, cache)
    pages[0][..., 0].view(torch.uint8).zero_()
    k = R.rows_of(pages[0], pages[2], torch.arange(kv, device="cuda"))
    q = (torch.rand(n, 2, dim, generator=g, device="cuda") + 1.0) * 2.0 ** -16
    q *= torch.randint(0, 2, q.shape, generator=g, device="cuda") * 2 - 1
    q[..., 0] = 1.0
    q = (q * 2.0 ** exponent).to(BF16)
    scale = 4.0 / float((q.double()[:, 0] @ k[:, 0].T).std())  # scores of a few
    out, lse, (want, mag, wlse), v = paged(scratch, pages, q, kv, scale=float(torch.tensor(scale, dtype=torch.float32)))
    check_attention(out, lse, want, mag, wlse, BF16, kv, float(v.abs().max()))


def test_rows_may_lie_in_any_order_that_keeps_them_apart():
    """Random strides: what overlaps is refused, all else is written, each row in its place."""
    r, g = random.Random(5), gen(53)
    turns, _ = S.rope_turns(16, 1e4)
    seen = [0, 0]
    for _ in range(300):
        tokens, heads = r.randint(1, 6), r.randint(1, 6)
        ts, hs = r.randint(0, 12) * 8, r.randint(0, 12) * 8
        at = [t * ts + h * hs for t in range(tokens) for h in range(heads)]
        apart = all(abs(a - b) >= 16 for i, a in enumerate(at) for b in at[:i])
        seen[apart] += 1
        space = torch.zeros(max(at) + 16, device="cuda")
        out = space.as_strided((tokens, heads, 16), (ts, hs, 1))
        x = randn(g, tokens, heads, 16)
        pos = torch.arange(tokens, dtype=torch.int32, device="cuda") * 77
        if apart:
            want = S.rope_rows(torch.empty_like(x), x, pos, turns)
            assert torch.equal(S.rope_rows(out, x, pos, turns), want)
            assert space.count_nonzero() == want.count_nonzero()
        else:
            with pytest.raises(S.XpError, match="overlap"):
                S.rope_rows(out, x, pos, turns)
    assert min(seen) > 30


@pytest.mark.parametrize("cache", [F16, I8])
@pytest.mark.parametrize("n", [1, 40])
def test_paged_lengths_up_to_the_last_whole_tile_below_2_31(scratch, cache, n):
    """The last tile of 2^31 - 256 keys is read as any other; what lies beyond is
    reported as past the table."""
    g = gen(55)
    page, dim = 8, 64
    pages = make_cache(g, 3, page, 1, dim, cache)
    table = torch.zeros(1, (1 << 28) - 1, dtype=torch.int32, device="cuda")
    table[0, ((1 << 31) - 256) // page - 20:] = 1  # the last keys of the long sequence: page 1, the others page 0
    q = randn(g, n, 2, dim, dtype=F16)

    def run(t, kv):
        out = torch.full_like(q, float("nan"))
        S.attention_paged(out, q, *pages, t, ints([kv]), ints([0, n]), n, scratch, window=250)
        return out, S.error_word(scratch)

    short = torch.zeros(1, 64, dtype=torch.int32, device="cuda")
    short[0, 44:] = 1
    want, word = run(short, 512)
    assert word == 0
    for kv, reported in (((1 << 31) - 256, 0), ((1 << 31) - 255, 1), ((1 << 31) - 8, 1)):
        out, word = run(table, kv)
        assert word == reported and torch.equal(out, want)
