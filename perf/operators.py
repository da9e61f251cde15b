"""Cases and plain forms of the paged-serving operators (xpose_b200.serving).

Four operators, used together when many sequences share one paged cache:

  rope    rotary positions on rows of heads (half or interleaved pairs, the
          whole head or its first `rot` values, frequencies stretched for long
          contexts), forward or inverse
  cache   keys and values quantised as they are written into pages (keys
          rotated on the way where `rot` is set), and read back
  packed  causal attention over whole prompts of different lengths, packed one
          after the other, with grouped heads and an optional sliding window
  paged   attention of each sequence's newest tokens (one to thousands) over
          its pages, which include those tokens

With `own` false `run` computes them by elementary torch operations in fp32;
with `own` true it calls xpose_b200.serving.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "fp8": 1}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}  # largest code of each 8-bit type
FLOOR = 2.0 ** -100                  # smallest row maximum that is told from zero
SCRATCH = 48 << 20                   # workspace of the two attentions


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _rope(**c):
    return {"op": "rope", "tokens": 64, "heads": 4, "dim": 256, "rot": 256, "layout": "half", "dtype": "f16",
            "theta": 1e6, "stretch": "none", "factor": 1.0, "inverse": False, "fused": False, "far": 4096, **c}


def _cache(**c):
    return {"op": "cache", "tokens": 64, "back": 64, "kv_heads": 1, "dim": 256, "page": 16, "cache": "int8",
            "dtype": "f16", "rot": 0, "layout": "half", "theta": 1e6, "far": 4096, **c}


def _packed(**c):
    return {"op": "packed", "batch": 4, "lo": 1, "hi": 128, "heads": 4, "kv_heads": 1, "dim": 256, "window": 0,
            "dtype": "f16", "fused": False, **c}


def _paged(**c):
    return {"op": "paged", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 4096, "kv_hi": 4096, "heads": 4,
            "kv_heads": 1, "dim": 256, "page": 16, "cache": "f16", "dtype": "f16", "window": 0, "idle": 0, **c}


def listed():
    return [
        # one decode step of a full batch (64 sequences) of the 4-head, 256-wide model: latency
        dict(_rope(tokens=64), name="rope step"),
        # a long prompt's queries inside fused q|k|v rows, half of each head, adjacent pairs, stretched context
        dict(_rope(tokens=16381, heads=32, dim=128, rot=64, layout="interleaved", dtype="bf16", stretch="parts",
                   factor=8.0, fused=True, far=131072), name="rope prompt"),
        # the new token of 64 sequences written in 8 bits with rotated keys, and those rows read again
        dict(_cache(tokens=64, back=64, rot=256), name="cache step int8"),
        # a chunk of prompt written in fp8, and four times as many rows brought back for reuse
        dict(_cache(tokens=8191, back=32768, kv_heads=8, dim=128, page=64, cache="fp8", dtype="bf16"),
             name="cache prompt fp8"),
        # short chat turns, one of a single token, over the 512-position sliding window of a local layer
        dict(_packed(batch=7, lo=1, hi=1100, window=512, dtype="bf16"), name="packed turns"),
        # a batch of prompts of ragged lengths, grouped heads
        dict(_packed(batch=12, lo=33, hi=2048, heads=32, kv_heads=8, dim=128, fused=True), name="packed ragged"),
        # one long prompt on a global layer of the 4-head, 256-wide model
        dict(_packed(batch=1, lo=8192, hi=8192, dtype="bf16"), name="packed long"),
        # a lone user's next token at position 4095
        dict(_paged(), name="paged one token"),
        # a server's decode step: 64 users of very different context lengths, some slots idle, fp8 pages
        dict(_paged(batch=64, kv_lo=64, kv_hi=16384, heads=32, kv_heads=8, dim=128, page=64, cache="fp8",
                    dtype="bf16", idle=8), name="paged step fp8"),
        # drafted tokens checked together (1 to 4 a sequence), narrow heads, int8 pages, sliding window
        dict(_paged(batch=16, q_hi=4, kv_lo=300, kv_hi=5000, heads=16, kv_heads=4, dim=64, page=32, cache="int8",
                    window=1024), name="paged drafts int8"),
        # prompt chunks of several users over the 4-head model's pages
        dict(_paged(batch=5, q_lo=37, q_hi=512, kv_lo=600, kv_hi=8192, cache="int8", dtype="bf16"),
             name="paged chunks int8"),
        # a long document's next chunk
        dict(_paged(batch=1, q_lo=2048, q_hi=2048, kv_lo=32768, kv_hi=32768, heads=16, kv_heads=2, dim=128, page=64,
                    cache="bf16", dtype="bf16"), name="paged document"),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))

    most = [work(c) for c in listed()]
    most = {op: {k: max(w[k] for c, w in zip(listed(), most) if c["op"] == op) for k in ("bytes", "flops")}
            for op in ("rope", "cache", "packed", "paged")}
    while True:
        op = rng.choice(["rope", "cache", "packed", "paged", "paged"])
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
        half = rng.choice(["f16", "bf16"])
        if op == "rope":
            stretch = rng.choice(["none", "linear", "base", "parts"])
            c = _rope(tokens=log(1, 16384), heads=heads, dim=dim, rot=dim // rng.choice([1, 1, 2, 4]),
                      layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["f16", "bf16", "f32"]),
                      theta=rng.choice([1e4, 5e5, 1e6]), stretch=stretch,
                      factor=1.0 if stretch == "none" else rng.choice([2.0, 4.0, 8.0, 32.0]),
                      inverse=rng.random() < 0.25, fused=rng.random() < 0.5, far=log(64, 1 << 20))
        elif op == "cache":
            tokens = log(1, 8192)
            c = _cache(tokens=tokens, back=min(32768, tokens + log(1, 32768) - 1), kv_heads=kv_heads, dim=dim,
                       page=rng.choice([8, 16, 32, 64, 128]), cache=rng.choice(["int8", "fp8", half]), dtype=half,
                       rot=rng.choice([0, dim, dim // 2]), layout=rng.choice(["half", "interleaved"]),
                       far=log(4096, 1 << 17))
        elif op == "packed":
            hi = log(1, 8192)
            c = _packed(batch=log(1, 24), lo=log(1, hi), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim,
                        window=rng.choice([0, 0, log(1, 2048)]), dtype=half, fused=rng.random() < 0.5)
            if heads * sum(_lens(c)) ** 2 > 1.2e9:  # the plain form's scores: at most 5 GB of them
                continue
        else:
            q_hi = rng.choice([1, 1, 4, log(1, 2048)])
            kv_hi = log(q_hi, 32768)
            c = _paged(batch=log(1, 64), q_lo=log(1, q_hi), q_hi=q_hi, kv_lo=log(1, kv_hi), kv_hi=kv_hi, heads=heads,
                       kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 32, 64, 128]),
                       cache=rng.choice([half, "int8", "fp8"]), dtype=half,
                       window=rng.choice([0, 0, log(1, 4096)]), idle=rng.choice([0, 3]))
            if max(c["batch"] * kv_hi * kv_heads * dim, c["batch"] * heads * q_hi * kv_hi) > 1.2e9:
                continue
        w = work(c)
        if w["bytes"] <= most[op]["bytes"] and w["flops"] <= most[op]["flops"]:
            return c


def _spread(n, lo, hi, salt):
    """n lengths between lo and hi, even over the logarithm, the largest first; the same for every seed."""
    r = random.Random(salt * 1000003 + n * 131 + lo * 17 + hi)
    return [hi] + [min(hi, max(lo, int(math.exp(r.uniform(math.log(lo), math.log(hi + 0.5)))))) for _ in range(n - 1)]


def _lens(c):
    return _spread(c["batch"], c["lo"], c["hi"], 1)


def _paged_lens(c):
    """(new tokens, tokens in the cache with them) of each sequence; every `idle`-th slot has none of either."""
    q = _spread(c["batch"], c["q_lo"], c["q_hi"], 2)
    kv = [max(a, b) for a, b in zip(q, _spread(c["batch"], c["kv_lo"], c["kv_hi"], 3))]
    gone = [c["idle"] and i % c["idle"] == c["idle"] - 1 for i in range(c["batch"])]
    return [0 if g else a for g, a in zip(gone, q)], [0 if g else a for g, a in zip(gone, kv)]


def _pairs(q, kv, window):
    """(query, key) pairs that one head's mask leaves: query i of q sits at kv - q + i."""
    if not q:
        return 0
    if not window:
        return q * (kv - q) + q * (q + 1) // 2
    full = max(0, min(q, kv - window + 1 if kv >= window else 0))  # queries that see a whole window
    rest = q - full
    return full * window + rest * (kv - q) + rest * (rest + 1) // 2


def work(c):
    op, size = c["op"], SIZE[c["dtype"]]
    if op == "rope":  # the rotated values in and out; the rest of the head is copied with them
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * size + 8 * c["tokens"], "flops": 3 * n * c["rot"]}
    if op == "cache":
        held = c["dim"] * SIZE[c["cache"]] + (4 if c["cache"] in TOP else 0)
        n, back = 2 * c["tokens"] * c["kv_heads"], 2 * c["back"] * c["kv_heads"]
        return {"bytes": (n + back) * (c["dim"] * size + held) + 8 * (c["tokens"] + c["back"]),
                "flops": 3 * n * c["dim"] + back * c["dim"] + (3 * n // 2) * c["rot"]}
    if op == "packed":
        lens = _lens(c)
        rows = sum(lens) * c["dim"] * size
        return {"bytes": rows * 2 * (c["heads"] + c["kv_heads"]),
                "flops": 4 * c["heads"] * c["dim"] * sum(_pairs(n, n, c["window"]) for n in lens)}
    q, kv = _paged_lens(c)
    seen = [min(b, a + c["window"] - 1) if c["window"] else b for a, b in zip(q, kv)]
    held = c["dim"] * SIZE[c["cache"]] + (4 if c["cache"] in TOP else 0)
    return {"bytes": 2 * sum(seen) * c["kv_heads"] * held + 2 * sum(q) * c["heads"] * c["dim"] * size
            + 4 * sum(-(-n // c["page"]) for n in seen),
            "flops": 4 * c["heads"] * c["dim"] * sum(_pairs(a, b, c["window"]) for a, b in zip(q, kv))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
ORIGINAL = 8192          # context that a stretched table was made for
SLOW, FAST = 1.0, 32.0   # turns over it below which a frequency is divided, above which it is kept


def _frequencies(rot, theta, stretch, factor):
    """Radians a position for each pair, and the factor on the rotated values."""
    if stretch == "base":
        theta = theta * factor ** (rot / (rot - 2))
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if stretch == "linear":
        f = [x / factor for x in f]
    if stretch == "parts":
        keep = [min(1.0, max(0.0, (ORIGINAL * x / (2 * math.pi) - SLOW) / (FAST - SLOW))) for x in f]
        f = [x * (k + (1 - k) / factor) for x, k in zip(f, keep)]
    return f, 0.1 * math.log(factor) + 1.0 if stretch == "parts" else 1.0


def _turns(f):
    """Frequencies as 64-bit fractions of a turn a position."""
    t = [int(math.ldexp(x / (2 * math.pi), 64)) & (2 ** 64 - 1) for x in f]
    return torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in t], dtype=torch.int64, device="cuda")


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _fused(g, tokens, heads, kv_heads, dim, dtype, fused):
    """q, k and v of each token: slices of one row of a q|k|v product, or tensors of their own."""
    if fused:
        x = _normal(g, (tokens, heads + 2 * kv_heads, dim), dtype)
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    return tuple(_normal(g, (tokens, n, dim), dtype) for n in (heads, kv_heads, kv_heads))


def _pages(g, pages, kv_heads, page, dim, cache):
    """Pages as earlier tokens left them: codes with a scale a row, or 16-bit values."""
    s = {}
    for n in "kv":
        if cache in TOP:
            x = torch.randn((pages, kv_heads, page, dim), generator=g, device="cuda") * (TOP[cache] / 4)
            x = x.clamp_(-TOP[cache], TOP[cache])
            s[n + "_pages"] = (x.round_() if cache == "int8" else x).to(CODES[cache])
            del x
            spread = torch.rand((pages, kv_heads, page), generator=g, device="cuda") + 0.5
            s[n + "_scale"] = spread * (4 / TOP[cache])
        else:
            s[n + "_pages"] = _normal(g, (pages, kv_heads, page, dim), TYPES[cache])
            s[n + "_scale"] = None
    return s


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s, dtype = case, {"case": case}, TYPES[case["dtype"]]
    if c["op"] in ("rope", "cache"):
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda", dtype=torch.int32)
    if c["op"] == "rope":
        f, s["magnitude"] = _frequencies(c["rot"], c["theta"], c["stretch"], c["factor"])
        s["turns"] = _turns(f)
        s["x"] = _fused(g, c["tokens"], c["heads"], 1, c["dim"], dtype, c["fused"])[0]
        s["out"] = torch.empty((c["tokens"], c["heads"], c["dim"]), dtype=dtype, device="cuda")
    elif c["op"] == "cache":
        pages = -(-c["back"] // c["page"]) + 3
        s |= _pages(g, pages, c["kv_heads"], c["page"], c["dim"], c["cache"])
        s["k"] = _normal(g, (c["tokens"], c["kv_heads"], c["dim"]), dtype)
        s["v"] = _normal(g, (c["tokens"], c["kv_heads"], c["dim"]), dtype, 0.3)
        # rows read: whole pages in the order of a block table; rows written: some of those
        order = torch.randperm(pages, generator=g, device="cuda")
        rows = (order[:, None] * c["page"] + torch.arange(c["page"], device="cuda")).reshape(-1)
        s["back_slots"] = rows[: c["back"]].contiguous()
        s["slots"] = s["back_slots"][torch.randperm(c["back"], generator=g, device="cuda")[: c["tokens"]]].contiguous()
        s["turns"] = _turns(_frequencies(c["rot"], c["theta"], "none", 1.0)[0]) if c["rot"] else None
        for n in ("k_out", "v_out"):
            s[n] = torch.empty((c["back"], c["kv_heads"], c["dim"]), dtype=dtype, device="cuda")
    elif c["op"] == "packed":
        lens = _lens(c)
        s["starts"] = _starts(lens)
        s["q"], s["k"], s["v"] = _fused(g, sum(lens), c["heads"], c["kv_heads"], c["dim"], dtype, c["fused"])
        s["out"] = torch.empty((sum(lens), c["heads"], c["dim"]), dtype=dtype, device="cuda")
        s["scratch"] = torch.zeros(SCRATCH, dtype=torch.uint8, device="cuda")
    else:
        q, kv = _paged_lens(c)
        s["starts"], s["kv_lens"], s["q_most"] = _starts(q), _ints(kv), max(q)
        held = [-(-n // c["page"]) for n in kv]
        pages = sum(held) + 2
        s |= _pages(g, pages, c["kv_heads"], c["page"], c["dim"], c["cache"])
        order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
        at = torch.arange(max(held), device="cuda")[None] + _ints([0] + held[:-1], torch.int64).cumsum(0)[:, None]
        has = torch.arange(max(held), device="cuda")[None] < _ints(held)[:, None]
        s["table"] = torch.where(has, order[at.clamp(max=pages - 1)], -1).to(torch.int32)
        s["q"] = _normal(g, (sum(q), c["heads"], c["dim"]), dtype)
        s["out"] = torch.empty_like(s["q"])
        s["scratch"] = torch.zeros(SCRATCH, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        from xpose_b200 import serving

        if c["op"] == "rope":
            serving.rope_rows(s["out"], s["x"], s["positions"], s["turns"], layout=c["layout"],
                              magnitude=s["magnitude"], inverse=c["inverse"])
            return s["out"]
        if c["op"] == "cache":
            pages = s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]
            serving.kv_write(*pages, s["k"], s["v"], s["slots"], positions=s["positions"] if c["rot"] else None,
                             turns=s["turns"], layout=c["layout"])
            serving.kv_read(*pages, s["k_out"], s["v_out"], s["back_slots"])
            return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if c["op"] == "packed":
            serving.attention_packed(s["out"], s["q"], s["k"], s["v"], s["starts"], s["scratch"],
                                     window=c["window"])
            return s["out"]
        serving.attention_paged(s["out"], s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"],
                                s["kv_lens"], s["starts"], s["q_most"], s["scratch"], window=c["window"])
        return s["out"]
    dtype = TYPES[c["dtype"]]
    if c["op"] == "rope":
        x = _rotated(s["x"].float(), s["positions"], s["turns"], c["layout"], s["magnitude"], c["inverse"])
        return x.to(dtype)
    if c["op"] == "cache":
        k = s["k"].float()
        k = _rotated(k, s["positions"], s["turns"], c["layout"], 1.0, False) if c["rot"] else k
        _write(s["k_pages"], s["k_scale"], s["slots"], k, c["cache"])
        _write(s["v_pages"], s["v_scale"], s["slots"], s["v"].float(), c["cache"])
        return {"k": _read(s["k_pages"], s["k_scale"], s["back_slots"]).to(dtype),
                "v": _read(s["v_pages"], s["v_scale"], s["back_slots"]).to(dtype),
                "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "packed":
        n = s["q"].shape[0]
        at = torch.arange(n, device="cuda", dtype=torch.int32)
        seq = torch.bucketize(at, s["starts"][1:], right=True)
        seen = (seq[:, None] == seq[None]) & (at[None] <= at[:, None])
        if c["window"]:
            seen &= at[None] > at[:, None] - c["window"]
        o = _attended(s["q"].float().transpose(0, 1)[None], s["k"].float().transpose(0, 1)[None],
                      s["v"].float().transpose(0, 1)[None], seen[None])
        return o[0].transpose(0, 1).contiguous().to(dtype)
    # paged: sequences side by side, padded to the longest
    q, batch, most = s["q"], c["batch"], s["q_most"]
    at = torch.arange(q.shape[0], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(at, s["starts"][1:], right=True)
    col = at - s["starts"][seq]
    wide = torch.zeros((batch, most, c["heads"], c["dim"]), device="cuda")
    wide[seq, col] = q.float()
    rows = (s["table"].clamp(min=0).long()[:, :, None] * c["page"] + torch.arange(c["page"], device="cuda"))
    rows = rows.reshape(-1)
    shape = (batch, -1, c["kv_heads"], c["dim"])
    k = _read(s["k_pages"], s["k_scale"], rows).reshape(shape).transpose(1, 2)
    v = _read(s["v_pages"], s["v_scale"], rows).reshape(shape).transpose(1, 2)
    key = torch.arange(k.shape[2], device="cuda", dtype=torch.int32)[None, None]
    first = s["kv_lens"] - (s["starts"][1:] - s["starts"][:-1])
    pos = (first[:, None] + torch.arange(most, device="cuda", dtype=torch.int32))[:, :, None]
    seen = (key <= pos) & (key < s["kv_lens"][:, None, None])
    if c["window"]:
        seen &= key > pos - c["window"]
    return _attended(wide.transpose(1, 2), k, v, seen).transpose(1, 2)[seq, col].to(dtype)


def _attended(q, k, v, seen):
    """Softmax attention: q [B, heads, rows, dim], k and v [B, kv heads, keys, dim], seen [B, rows, keys]."""
    b, heads, rows, dim = q.shape
    group = heads // k.shape[1]
    p = torch.matmul(q.reshape(b, -1, group * rows, dim), k.transpose(2, 3)).mul_(dim ** -0.5)
    p = p.view(b, -1, group, rows, k.shape[2])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, -1, group * rows, k.shape[2]), v).view(b, -1, group, rows, dim)
    return (o / torch.where(total == 0, 1.0, total)).reshape(b, heads, rows, dim)


def _rotated(x, positions, turns, layout, magnitude, inverse):
    """x [tokens, heads, dim] with the first 2 * len(turns) values of each head rotated by the position's angles."""
    part = (positions.long()[:, None] * turns) >> 32  # of a turn, in 2^-32: whole turns fall out by themselves
    angle = part.float() * (2 * math.pi / 2 ** 32)
    cos, sin = angle.cos()[:, None] * magnitude, angle.sin()[:, None] * (-magnitude if inverse else magnitude)
    n = turns.numel()
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., 2 * n:]), -1)
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((r, x[..., 2 * n:]), -1)


def _write(pages, scale, slots, x, cache):
    """x [tokens, kv heads, dim] into the rows `slots` of pages [pages, kv heads, page, dim]."""
    page, row = slots // pages.shape[2], slots % pages.shape[2]
    if cache not in TOP:
        pages[page, :, row] = x.to(pages.dtype)
        return
    top = x.abs().amax(-1).clamp(min=FLOOR)
    most = torch.full_like(top, TOP[cache])
    code = x * (most / top)[..., None]
    if cache == "int8":
        pages[page, :, row] = code.round().clamp(-127, 127).to(torch.int8)
    else:  # fp8 has no indexed stores: write the bytes
        pages.view(torch.uint8)[page, :, row] = code.to(torch.float8_e4m3fn).view(torch.uint8)
    scale[page, :, row] = top / most


def _read(pages, scale, slots):
    """The fp32 values of the rows `slots`: [rows, kv heads, dim]."""
    page, row = slots // pages.shape[2], slots % pages.shape[2]
    if scale is None:
        return pages[page, :, row].float()
    if pages.dtype == torch.int8:
        x = pages[page, :, row].float()
    else:
        x = pages.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn).float()
    return x * scale[page, :, row][..., None]


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotation(x, positions, c, stretch, factor, inverse):
    f, magnitude = _frequencies(c["rot"], c["theta"], stretch, factor)
    angle = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda")
    z = torch.polar(torch.full_like(angle, magnitude), -angle if inverse else angle)[:, None]
    n, y = c["rot"] // 2, x.double().clone()
    first = slice(0, n) if c["layout"] == "half" else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if c["layout"] == "half" else slice(1, 2 * n, 2)
    w = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _exact_head(q, k, v, kv, window, scale):
    """One sequence and one head: q [n, dim] at positions kv - n .. kv - 1, k and v [kv, dim]."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for a in range(0, q.shape[0], 4096):
        rows = q[a:a + 4096].double()
        pos = torch.arange(a, a + rows.shape[0], device="cuda") + kv - q.shape[0]
        last = kv - q.shape[0] + a + rows.shape[0]
        from_ = max(0, kv - q.shape[0] + a - window + 1) if window else 0
        key = torch.arange(from_, last, device="cuda")
        t = (rows @ k[from_:last].double().T) * scale
        off = key[None] > pos[:, None]
        if window:
            off |= key[None] <= pos[:, None] - window
        t[off] = -math.inf
        out[a:a + 4096] = torch.softmax(t, -1) @ v[from_:last].double()
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        return _exact_rotation(s["x"], s["positions"], c, c["stretch"], c["factor"], c["inverse"])
    if c["op"] == "cache":
        got = {}
        for n in "kv":
            pages, scale, x = s[n + "_pages"], s[n + "_scale"], s[n].double()
            if n == "k" and c["rot"]:
                x = _exact_rotation(x, s["positions"], c, "none", 1.0, False)
            held = pages.float().double() * (1.0 if scale is None else scale.double()[..., None])
            at = s["slots"] // c["page"], slice(None), s["slots"] % c["page"]
            if c["cache"] in TOP:
                unit = x.abs().amax(-1).clamp(min=FLOOR) / TOP[c["cache"]]
                code = x / unit[..., None]
                if c["cache"] == "int8":
                    code = torch.round(code)
                else:  # three bits after the leading one, steps of 2^-9 below 2^-6
                    step = torch.exp2(torch.floor(torch.log2(code.abs().clamp(min=2.0 ** -6))) - 3)
                    code = torch.round(code / step) * step
                held[at] = code * unit[..., None]
                units = scale.double()
                units[at] = unit
                got[n + "_scale"] = units
            else:
                held[at] = x.to(TYPES[c["cache"]]).double()
                got[n + "_scale"] = None
            got[n] = held[s["back_slots"] // c["page"], :, s["back_slots"] % c["page"]]
        return got
    group, scale = c["heads"] // c["kv_heads"], c["dim"] ** -0.5
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q_lens, kv_lens = (_lens(c), _lens(c)) if c["op"] == "packed" else _paged_lens(c)
    at = 0
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if not n:
            continue
        if c["op"] == "packed":
            k, v = s["k"][at:at + n], s["v"][at:at + n]
        else:
            used = s["table"][b, : -(-kv // c["page"])].long()
            k, v = ((s[m + "_pages"].view(torch.uint8)[used].view(s[m + "_pages"].dtype).double()
                     * (1.0 if s[m + "_scale"] is None else s[m + "_scale"][used].double()[..., None]))
                    .transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[:kv] for m in "kv")
        for h in range(c["heads"]):
            out[at:at + n, h] = _exact_head(s["q"][at:at + n, h], k[:, h // group], v[:, h // group], kv,
                                            c["window"], scale)
        at += n
    return out
