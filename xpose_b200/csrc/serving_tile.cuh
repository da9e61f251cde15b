// Attention of many rows on the 5th-generation tensor cores: whole prompts,
// and chunks of new tokens over pages.
//
// One CTA an SM works through tiles of 128 * NQ rows. The rows of a tile are
// whole tokens times the `group` query heads that share one kv head, so K and
// V are read once for all of them. For each 128 keys:
//   S = Q K^T        tcgen05.mma, operands in shared memory, S in TMEM
//   P = 2^(S - m)    one thread a row, S and P in TMEM, P in 16 bits over S
//   O += P V         tcgen05.mma with P from TMEM, O in TMEM
// m is the row's maximum when it was last set: it follows a new maximum only
// when that is more than 2^8 away (O and l are then scaled), so O is seldom
// touched between two products; P up to 2^8 loses nothing in either type.
//
// dim 64 and 128: two row tiles (NQ = 2) share every K and V tile, and the
// softmax of one runs beside the products of the other. dim 256: O fills half
// of TMEM, so one row tile (NQ = 1) with two S buffers; the products of one
// key tile run beside the softmax of the next.
//
// K and V move in pieces of a tile (dim 256: of half a tile, K by dims and V by
// keys) through one ring, so a ring slot is free again as soon as its piece is
// multiplied. 16-bit rows come by TMA, a box a page, straight into the
// 128-byte swizzled layouts of the tensor core; a page that a tile must not
// touch is read past the end of the tensor, which gives zeros. What a tile's
// last page or the next sequence holds past the tile's keys must not be
// multiplied even by 0 (it may be NaN): in the few V tiles where some row does
// not see some key, loader threads put zeros there, and take infinities and
// NaN of v out (codes of NaN, too); those go to the rows that do see them at the end. 8-bit codes
// are turned into exact 16-bit values by the loader threads; their scales
// never touch them: with t_ij = s_ij ks_j + log2 vs_j the weight that
// multiplies v's code is 2^(t - m), and l adds 2^(t - m) / vs_j. A weight is
// then rounded relative to the largest contribution, whatever the scales. Rows
// whose scale is zero or next to it have no such weight: their codes are read as
// zeros with a scale of 1.
//
// Work is split evenly: every CTA takes the same number of (row tile, key
// tile) units, so the last tile of a call does not run alone. A row tile that
// two or more CTAs share leaves partial sums (O, m, l) that a second, small
// launch joins in a fixed order.
//
// Measured, a call (and its kernels alone, replayed from a graph): 2048 tokens over
// 32768 keys, 16 / 2 heads of 128, bf16: 482 us, 1.11 PFLOP/s (408 to 492 us as the
// power limit has it), bound by the softmax of a row tile, which its own products
// wait for; a prompt of 8192, 4 / 1 heads of 256: 154 us, 0.89 PFLOP/s (143 to 151), bound
// by shared memory (320 KB of operands and copies for 2048 cycles of products); 12
// prompts of 33 to 2048, 32 / 8 heads of 128, fp16: 123 us, 0.58 PFLOP/s (107 to 110); 5
// chunks of 37 to 512 over int8 pages, 4 / 1 heads of 256: 52 us (50).
#pragma once
#include <cuda.h>

#include "serving_attn.cuh"
#include "tk_primitives.cuh"

namespace xp {

constexpr int AT_KEYS = 128;        // keys of a tile
constexpr uint32_t AT_COST = 2;     // what a row tile costs besides its key tiles, in key tiles
constexpr uint32_t AT_SHIFT = 7;    // log2 AT_KEYS
constexpr uint32_t AT_NONE = 0xFFFFFFFFu;
constexpr uint32_t AT_SPIN_LIMIT = 1u << 20;
constexpr uint32_t AT_MAX_CTAS = 180;   // partial slots that the scratch holds
constexpr uint32_t AT_MAX_BATCH = 8192;   // sequences whose tile counts fit in shared memory

template <class T, class C, int W> struct AtCfg {
    static constexpr int D = 64 * W;
    static constexpr bool Q8 = sizeof(C) == 1;
    static constexpr int NQ = W == 4 ? 1 : 2;     // row tiles of a CTA
    static constexpr int NB = 2 / NQ;             // S buffers of a row tile
    static constexpr int ROWS = 128 * NQ;
    static constexpr int LAG = NB;                // K runs this many tiles ahead of V
    static constexpr int NP = W == 4 ? 2 : 1;     // pieces of a K (or V) tile
    static constexpr int PIECE = W * 16384 / NP;  // bytes of one, and of a ring slot
    static constexpr int KB = W / NP;             // blocks of 64 dims of a K piece
    static constexpr int VKEYS = AT_KEYS / NP;    // keys of a V piece
    static constexpr int NSLOT = W == 1 ? 10 : Q8 ? 4 : 5;
    static constexpr int NSTAGE = W == 1 ? 8 : 4; // tiles whose row numbers and scales are kept
    static constexpr int NLD = Q8 && W == 4 ? 2 : 1;  // loader warpgroups
    static constexpr int THREADS = 128 * NQ + 128 * NLD + 128;
    // registers of a softmax, a loader and the last warpgroup: THREADS / 128 shares of the launch's.
    // Loaders of 128-wide e4m3 heads get 96: with 80 the look for codes of NaN spills. Prompt chunks
    // take 139 us with 96, 148 with 80; int8 153 and 140, 64-wide heads of both 65 and 61
    static constexpr bool MORE = W == 2 && std::is_same_v<C, fp8c>;
    static constexpr int R_SOFT = MORE ? 176 : NQ == 2 ? 184 : NLD == 2 ? 208 : 232;
    static constexpr int R_LOAD = MORE ? 96 : NQ == 2 ? 80 : NLD == 2 ? 104 : 136;
    static constexpr int R_REST = NQ == 2 ? 64 : NLD == 2 ? 96 : 136;
    static_assert(NQ * R_SOFT + NLD * R_LOAD + R_REST <= THREADS / 128 * (65536 / THREADS / 8 * 8), "registers");
    // shared memory
    static constexpr int q_off = 0;
    static constexpr int ring_off = NQ * W * 16384;
    static constexpr int row_off = ring_off + NSLOT * PIECE;       // [NSTAGE][2][128] row numbers of k and v, 8-bit pages
    static constexpr int sc_off = row_off + (Q8 ? NSTAGE * 1024 : 0);  // [NSTAGE][3][128] floats, 8-bit pages
    static constexpr int bar_off = sc_off + (Q8 ? NSTAGE * 1536 : 0);
    static constexpr int smem = bar_off + 1024;                       // barriers, plan, row tiles, flags
};

struct AtWork {
    unsigned char* slots;   // partial sums: two of slot_bytes a CTA
    uint32_t* heads;        // [2 * CTAs][4]: kind, b, h, tile of each
    uint32_t slot_bytes;
    uint32_t head_step;     // packed: k and v heads a kv head apart in the tensor maps (0: one for all)
    uint32_t tile_tokens;   // tokens of a tile
    uint32_t sub_tokens;    // tokens of one of its NQ row tiles
    uint32_t least_units;   // units of a CTA, at least
    uint32_t split_over;    // whole tiles while none has more units, or more than an eighth of a CTA's
};
enum : uint32_t { AT_FULL = 0, AT_FIRST = 1, AT_MIDDLE = 2, AT_LAST = 3, AT_END = 4 };

// ---- tcgen05 ------------------------------------------------------------------
// Shared-memory operands: 128-byte swizzle (layout type 2), descriptor version
// 1, 1 KB between groups of 8 rows. Low half: address and leading offset.
XP_DEV uint32_t at_desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16); }
XP_DEV uint64_t at_desc(uint32_t lo) {
    return (uint64_t)lo | ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32);
}
XP_DEV bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
template <class T> XP_DEV uint32_t at_idesc(uint32_t n, bool b_mn) {
    const uint32_t f = std::is_same_v<T, bf16> ? 1u : 0u;
    return (1u << 4) | (f << 7) | (f << 10) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
XP_DEV void at_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
XP_DEV void at_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"(acc)
        : "memory");
}
XP_DEV void at_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
XP_DEV void at_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
XP_DEV void at_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
#define AT_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define AT_I8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
// 32 columns of the thread's TMEM lane
XP_DEV void at_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : AT_R8(r, 0), AT_R8(r, 8), AT_R8(r, 16), AT_R8(r, 24)
        : "r"(addr));
}
XP_DEV void at_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::AT_I8(r, 0),
        AT_I8(r, 8), AT_I8(r, 16), AT_I8(r, 24), "r"(addr)
        : "memory");
}
XP_DEV void at_ld16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : AT_R8(r, 0), AT_R8(r, 8)
        : "r"(addr));
}
XP_DEV void at_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::AT_I8(r, 0),
        AT_I8(r, 8), "r"(addr)
        : "memory");
}
XP_DEV void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
XP_DEV void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N> XP_DEV void at_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> XP_DEV void at_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

XP_DEV bool at_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
// Bounded: a wait that runs out reports it and lets every later wait of the
// CTA pass, so the kernel ends (with unspecified output). Once a CTA's warps
// have parted, each leaves on its own, so they meet in no barrier of threads
// before the last one.
XP_DEV void at_wait(uint32_t bar, uint32_t parity, volatile uint32_t* dead, uint32_t* err) {
    uint32_t it = 0;
    while (!at_try(bar, parity)) {
        if (*dead) return;
        if (++it > AT_SPIN_LIMIT) {
            *dead = 1;
            atomicOr(err, SERVE_ERR_WAIT);
            return;
        }
    }
}
// ... and after such a failure: for what is still on its way, whatever `dead` says
XP_DEV void at_wait_flight(uint32_t bar, uint32_t parity) {
    for (uint32_t it = 0; it < AT_SPIN_LIMIT && !at_try(bar, parity); ++it) {}
}
XP_DEV void at_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
XP_DEV float at_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 lanes at a time
XP_DEV float2 at_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
XP_DEV float2 at_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
XP_DEV float2 at_mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
// What brings a bf16 row whose largest exponent is e to [1, 2) (the largest
// rows to [2, 4); rows of zeros and subnormals stay)
XP_DEV float at_row_factor(uint32_t e) { return e ? __uint_as_float((uint32_t)max(254 - (int32_t)e, 1) << 23) : 1.0f; }
template <class T> XP_DEV uint32_t at_pack(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same_v<T, bf16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 4 codes -> 4 exact fp16 values
XP_DEV uint2 at_codes(uint32_t w, int8c) {
    // a biased code as the low bits of 2^10: 1024 + 128 + code, exact
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(reinterpret_cast<__half2&>(a), bias), y = __hsub2(reinterpret_cast<__half2&>(b), bias);
    return make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
}
XP_DEV uint2 at_codes(uint32_t w, fp8c) {
    uint32_t a, b;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"((uint16_t)w));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"((uint16_t)(w >> 16)));
    return make_uint2(a, b);
}
XP_DEV void at_tma(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
XP_DEV uint32_t at_lds(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
XP_DEV uint4 at_lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
XP_DEV void at_sts16(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

XP_DEV void at_stg32(void* p, uint4 a, uint4 b) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
                 "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

// ---- the split of the work --------------------------------------------------------
// Tile x of a sequence: tokens [x tt, ..), its key range [lo, hi) and the key
// tiles that cover it.
struct AtTile { int32_t lo, hi; uint32_t t0, n; };
XP_DEV AtTile at_tile(const Seq& s, uint32_t x, uint32_t tt, uint32_t window, uint32_t shift) {
    AtTile r;
    const int32_t first = (int32_t)s.nkv - (int32_t)s.nq;
    const uint32_t tok0 = x * tt, tok1 = min(tok0 + tt, s.nq);
    r.hi = max(first + (int32_t)tok1, 0);
    const int64_t lo = window ? (int64_t)first + tok0 + 1 - (int64_t)window : 0;
    r.lo = (int32_t)min(max(lo, (int64_t)0), (int64_t)r.hi);
    r.t0 = (uint32_t)r.lo >> shift;
    r.n = r.hi > r.lo ? (((uint32_t)r.hi - 1) >> shift) + 1 - r.t0 : 0;
    return r;
}

// Zeros for the rows of q that are in no sequence.
template <class T, int D> XP_DEV void at_clear(const ServeAttnArgs& a, uint32_t threads) {
    const uint32_t lo = (uint32_t)min(max(ld_now(a.starts), 0), (int32_t)a.tokens);
    const uint32_t hi = max((uint32_t)min(max(ld_now(a.starts + a.batch), 0), (int32_t)a.tokens), lo);
    const uint64_t n = (uint64_t)(lo + (a.tokens - hi)) * a.heads * (D / 8);
    for (uint64_t i = (uint64_t)blockIdx.x * threads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * threads) {
        const uint32_t d = (uint32_t)(i % (D / 8)) * 8, h = (uint32_t)(i / (D / 8) % a.heads);
        uint32_t tok = (uint32_t)(i / (D / 8) / a.heads);
        if (tok >= lo) tok += hi - lo;
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out.data) + (int64_t)tok * a.out.ts + (int64_t)h * a.out.hs + d) =
            make_uint4(0, 0, 0, 0);
        if (a.lse && d == 0) a.lse[(uint64_t)tok * a.heads + h] = -INFINITY;
    }
}

// Where a CTA starts in the list of units: head h, sequence b, tile x. A tile
// counts as its key tiles and AT_COST more, which come first.
struct AtPlan {
    uint32_t h, b, x, skip;   // skip: units of the first tile that earlier CTAs have
    int64_t todo;             // units from there; whole tiles: those that start within them
    bool split;
};

// 64-bit division, in 32 bits where both fit (a tenth of the time)
XP_DEV uint64_t at_div(uint64_t x, uint64_t y) {
    return (x | y) >> 32 ? x / y : (uint64_t)((uint32_t)x / (uint32_t)y);
}

XP_DEV uint32_t at_scan(uint32_t v, uint32_t* warp_sums, uint32_t nthreads, uint32_t& total) {
    // inclusive scan over the CTA; warp_sums: 32 words of shared memory
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= (uint32_t)o) v += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    uint32_t before = 0, sum = 0;
    for (uint32_t i = 0; i < nthreads / 32; ++i) {
        const uint32_t y = warp_sums[i];
        if (i < warp) before += y;
        sum += y;
    }
    total = sum;
    return v + before;
}

// Every thread of every CTA computes the same plan from the lengths alone.
// `ends`: shared memory for one word a sequence.
template <int THREADS>
XP_DEV void at_make_plan(const ServeAttnArgs& a, const AtWork& w, uint32_t* ends, uint32_t* sums, AtPlan* out) {
    const uint32_t tid = threadIdx.x;
    uint32_t tiles = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += THREADS) {
        const uint32_t b = b0 + tid;
        const uint32_t n = b < a.batch ? (seq_of(a, b).nq + w.tile_tokens - 1) / w.tile_tokens : 0;
        uint32_t sum;
        const uint32_t end = tiles + at_scan(n, sums, THREADS, sum);
        if (b < a.batch) ends[b] = end;
        tiles += sum;
    }
    __syncthreads();
    // units of a tile; its sequence by bisection
    auto units = [&](uint32_t i, uint32_t& b, uint32_t& x) {
        uint32_t lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (ends[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
        x = i - (lo ? ends[lo - 1] : 0);
        return at_tile(seq_of(a, b), x, w.tile_tokens, a.window, AT_SHIFT).n + AT_COST;
    };
    uint64_t all = 0;
    uint32_t most = 0, b = 0, x = 0, n = 0, end = 0;
    for (uint32_t i0 = 0; i0 < tiles; i0 += THREADS) {
        const uint32_t i = i0 + tid;
        n = i < tiles ? units(i, b, x) : 0;
        uint32_t sum;
        end = at_scan(n, sums, THREADS, sum);
        all += sum;
        most = max(most, n);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if ((tid & 31) == 0) sums[tid >> 5] = most;
    if (tid == 0) out->todo = 0;
    __syncthreads();
    for (int i = 0; i < THREADS / 32; ++i) most = max(most, sums[i]);
    __syncthreads();
    if (all == 0) return;
    // no CTA has less than a unit, so the parts of a tile are in consecutive CTAs
    const uint64_t total = all * a.kv_heads, c = blockIdx.x;
    const uint64_t g = min((uint64_t)gridDim.x, max(at_div(total, w.least_units), (uint64_t)1));
    if (c >= g) return;
    const uint64_t u0 = at_div(total * c, g), u1 = at_div(total * (c + 1), g);
    const bool split = most > max((uint64_t)w.split_over, at_div(total, 8 * g));
    if (u0 == u1) return;
    // the first tile of the range: split, the one that holds u0; else the
    // first that starts at or after it
    const uint32_t h0 = (uint32_t)at_div(u0, all);
    for (uint32_t h = h0; h < a.kv_heads && h <= h0 + 1; ++h) {
        uint64_t at = all * h;
        bool found = false;
        for (uint32_t i0 = 0; i0 < tiles && !found; i0 += THREADS) {
            const uint32_t i = i0 + tid;
            uint32_t sum = 0;
            if (tiles > THREADS) {  // else as in the loop above
                n = i < tiles ? units(i, b, x) : 0;
                end = at_scan(n, sums, THREADS, sum);
            }
            const uint64_t stop = at + end, begin = stop - n;
            const bool mine = n && (split ? begin <= u0 && u0 < stop : begin >= u0 && begin < u1);
            if (split) {
                if (mine) *out = AtPlan{h, b, x, (uint32_t)(u0 - begin), (int64_t)(u1 - u0), true};
                found = __syncthreads_or(mine);
            } else {
                // lowest index among the candidates
                const uint32_t best = __reduce_min_sync(0xffffffffu, mine ? i : AT_NONE);
                __syncthreads();
                if ((tid & 31) == 0) sums[tid >> 5] = best;
                __syncthreads();
                uint32_t low = AT_NONE;
                for (int j = 0; j < THREADS / 32; ++j) low = min(low, sums[j]);
                if (mine && i == low) *out = AtPlan{h, b, x, 0, (int64_t)(u1 - begin), false};
                found = low != AT_NONE;
                __syncthreads();
            }
            at += sum;
        }
        if (found || split) break;
    }
    __syncthreads();
}

// The part of a row tile that a CTA computes. One warp walks the CTA's range
// and hands these to the others through shared memory.
struct AtSeg {
    uint32_t h, b, x, kind;
    Seq s;
    int32_t lo, hi;     // the tile's keys
    int32_t p0;         // position of its first token
    uint32_t k0, n;     // first key tile and how many
};
struct AtWalk {
    AtPlan p;
    Seq s;
    uint32_t have;      // s is sequence have
    XP_DEV void start(const AtPlan& plan) { p = plan; have = AT_NONE; }
    __device__ bool next(const ServeAttnArgs& a, const AtWork& w, AtSeg& g) {
      for (;;) {
        if (p.todo <= 0) return false;
        for (;;) {
            if (have != p.b) {
                s = seq_of(a, p.b);
                have = p.b;
            }
            if (p.x * w.tile_tokens < s.nq) break;
            p.x = 0;
            if (++p.b == a.batch) {
                p.b = 0;
                if (++p.h >= a.kv_heads) return false;
            }
        }
        g.h = p.h;
        g.b = p.b;
        g.x = p.x;
        g.s = s;
        const AtTile t = at_tile(s, p.x, w.tile_tokens, a.window, AT_SHIFT);
        g.lo = t.lo;
        g.hi = t.hi;
        g.p0 = (int32_t)s.nkv - (int32_t)s.nq + (int32_t)(p.x * w.tile_tokens);
        // units [skip, skip + step) of the tile are these of its key tiles
        const uint32_t all = t.n + AT_COST;
        const uint32_t step = p.split ? (uint32_t)min((int64_t)(all - p.skip), p.todo) : all;
        const uint32_t from = max(p.skip, AT_COST) - AT_COST, to = max(p.skip + step, AT_COST) - AT_COST;
        g.kind = from == 0 ? (to == t.n ? AT_FULL : AT_FIRST) : (to == t.n ? AT_LAST : AT_MIDDLE);
        g.k0 = t.t0 + from;
        g.n = to - from;
        // no key tile falls to this CTA: a neighbour has the tile, or it has none
        const bool none = t.n ? to == from : p.skip != 0;
        p.todo -= step;
        p.skip = 0;
        ++p.x;
        if (!none) return true;
      }
    }
};

// The V rows of keys [k0, k0 + n) need a look: one lies outside the tile's
// keys, or some row of the tile does not see some of them.
XP_DEV bool at_look(const ServeAttnArgs& a, int32_t lo, int32_t hi, int32_t p0, uint32_t key, uint32_t n) {
    const int64_t k0 = (int64_t)key, k1 = k0 + n;
    return k0 < lo || k1 > hi || k1 > (int64_t)p0 + 1 || (a.window && k0 < (int64_t)hi - (int64_t)a.window);
}
// The top bits of bytes that are codes of NaN (all lower bits set)
XP_DEV uint32_t at_odd8(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// Bits 15 and 31: an infinity or NaN in either half (all exponent bits set, so
// one more carries out of them)
template <class T> XP_DEV uint32_t at_odd16(uint32_t w) {
    if constexpr (std::is_same_v<T, bf16>) return (w & 0x7F807F80u) + 0x00800080u;
    else return (w & 0x7C007C00u) + 0x04000400u;
}

template <class T, class C, int W>
__global__ void __launch_bounds__(AtCfg<T, C, W>::THREADS, 1)
attn_tile_kernel(const __grid_constant__ ServeAttnArgs a, const __grid_constant__ AtWork w,
                 const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap) {
    using G = AtCfg<T, C, W>;
    constexpr int D = G::D, NQ = G::NQ, NSLOT = G::NSLOT, NSTAGE = G::NSTAGE;
    // 8-bit codes are multiplied in fp16 whatever T is (a code costs half as
    // much to convert as in bf16): bf16 queries become fp16 in place
    constexpr uint32_t LAST = NQ * 4 + G::NLD * 4;  // first warp of the last warpgroup
    using M = std::conditional_t<G::Q8, __half, T>;
    constexpr bool RESCALE = G::Q8 && std::is_same_v<T, bf16>;
    constexpr bool ODD8 = std::is_same_v<C, fp8c>;  // 8-bit pages, and some codes are NaN
    // no static shared memory: the dynamic part then starts on a 1 KB boundary,
    // which the swizzled layouts need, without a byte lost
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t smb = smem_u32(sm);
    constexpr int NSEG = 4, NBAR = 4 * NSLOT + 16 + 2 * NSEG;
    struct Small {
        AtPlan plan;
        AtSeg segs[NSEG];
        uint32_t sums[32], bad[4], tmem, dead;
    };
    static_assert(NBAR * 8 + sizeof(Small) <= 1024 && NBAR * 8 % 8 == 0, "small data");
    Small& small = *reinterpret_cast<Small*>(sm + G::bar_off + NBAR * 8);
    AtPlan& s_plan = small.plan;
    uint32_t *const s_sums = small.sums, *const s_bad = small.bad;
    volatile uint32_t& s_dead = small.dead;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // barriers
    const uint32_t b_full = smb + G::bar_off;       // [NSLOT] a piece is in
    const uint32_t b_empty = b_full + NSLOT * 8;    // [NSLOT] ... multiplied
    // a piece that needs a look arrives on its own ring, in order: no wait of
    // the threads that look may skip a phase of its barrier
    const uint32_t b_raw = b_empty + NSLOT * 8;     // [NSLOT] a V piece to look over is in
    const uint32_t b_clean = b_raw + NSLOT * 8;     // [NSLOT] ... looked over
    const uint32_t b_q = b_clean + NSLOT * 8;       // [NQ] Q is in
    const uint32_t b_s = b_q + 16, b_p = b_s + 16;  // [2] S made, P made (by S buffer)
    const uint32_t b_o = b_p + 16;                  // [2] P V added, by S buffer
    const uint32_t b_seg = b_o + 16, b_free = b_seg + NSEG * 8;  // [NSEG] a row tile given, done with
    const uint32_t b_qfree = b_free + NSEG * 8;     // [NQ] Q multiplied for the last time
    const uint32_t b_qh = b_qfree + 16;             // [NQ] ... made fp16
    const uint32_t b_ph = b_qh + 16;                // [2] P's first 64 keys made (b_p: all), by S buffer
    const uint32_t b_end = b_ph + 16;               // products in flight after a failed wait
    const uint32_t b_rows = b_end + 8;              // 8-bit pages: row numbers and scales of a tile given to the loaders

    if (smb & 1023) {  // cannot be multiplied from
        pdl_wait();
        if (tid == 0) {
            w.heads[(2 * blockIdx.x) * 4] = w.heads[(2 * blockIdx.x + 1) * 4] = AT_FULL;  // nothing to join
            atomicOr(a.err, SERVE_ERR_WAIT);
        }
        return;
    }
    if (tid == 0) {
        uint64_t* m = reinterpret_cast<uint64_t*>(sm + G::bar_off);
        for (int i = 0; i < NSLOT; ++i) {
            mbar_init(m + i, G::Q8 ? 4 * G::NLD : 1);
            mbar_init(m + NSLOT + i, 1);
            mbar_init(m + 2 * NSLOT + i, 1);
            mbar_init(m + 3 * NSLOT + i, 4);
        }
        m += 4 * NSLOT;
        for (int i = 0; i < 2; ++i) {
            mbar_init(m + i, 1);
            mbar_init(m + 2 + i, 1);
            mbar_init(m + 4 + i, 4);
            mbar_init(m + 6 + i, 1);
        }
        for (int i = 0; i < NSEG; ++i) {
            mbar_init(m + 8 + i, 1);
            mbar_init(m + 8 + NSEG + i, NQ * 4 + G::NLD * 4 + 2);
        }
        for (int i = 0; i < 7; ++i) mbar_init(m + 8 + 2 * NSEG + i, i >= 2 && i < 6 ? 4 : 1);
        mbar_init(m + 15 + 2 * NSEG, 4 * G::NLD);
        fence_mbar_init();
        s_dead = 0;
        for (int i = 0; i < 4; ++i) s_bad[i] = 0;
    }
    if (warp == LAST) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&small.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if constexpr (G::Q8) {
        // after a failed wait a loader may meet row numbers that were never given: no row
        for (uint32_t i = tid; i < NSTAGE * 256; i += G::THREADS)
            *reinterpret_cast<uint32_t*>(sm + G::row_off + i * 4) = AT_NONE;
    }
    pdl_wait();  // everything above may run under the kernel before this one
    at_clear<T, D>(a, G::THREADS);
    at_make_plan<G::THREADS>(a, w, reinterpret_cast<uint32_t*>(sm), s_sums, &s_plan);
    fence_proxy_async();  // the plan's words before the copies of Q that take their place
    at_fence_before();
    __syncthreads();
    at_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = small.tmem;
    uint32_t* const err = a.err;
    // the next row tile of this CTA: given to every role in turn
    uint32_t seg = 0;
    auto take = [&]() -> const AtSeg& {
        at_wait(b_seg + 8 * (seg % NSEG), (seg / NSEG) & 1, &s_dead, err);
        return small.segs[seg % NSEG];
    };
    auto done = [&]() {
        __syncwarp();
        if (lane == 0) at_arrive(b_free + 8 * (seg % NSEG));
        ++seg;
    };

    if (warp < NQ * 4) {
        // ------------------------------ softmax ------------------------------
        at_regs_up<G::R_SOFT>();
        const uint32_t wg = warp >> 2, row = tid & 127;
        const uint32_t lanes = (warp & 3) * 32 << 16;
        const uint32_t o_tm = tmem + lanes + 256 + wg * D;
        if (tid == 0) {
            w.heads[(2 * blockIdx.x) * 4] = AT_FULL;
            w.heads[(2 * blockIdx.x + 1) * 4] = AT_FULL;
        }
        const uint32_t qrow0 = wg * w.sub_tokens;  // first token of this row tile in its CTA's tile
        // Phases are told apart by their parity alone, so a wait must come neither
        // before the phase ahead of its own has ended nor after the one behind it.
        // b_o: the product of the tile NB earlier, whose P shares this S buffer, ended
        // before S was made there (one thread issues and commits them in this order),
        // so no wait is spent on it: in front of the scores it took up to a tenth. The
        // next one on the buffer needs this warp's P. s_phase, o_phase: a bit for each
        // S buffer
        uint32_t stage = 0, s_phase = 0, o_phase = 0, q_phase = 0;
        auto take_o = [&](uint32_t buf) {
            at_wait(b_o + 8 * buf, o_phase >> buf & 1, &s_dead, err);
            o_phase ^= 1u << buf;
        };
        for (;; done()) {
            const AtSeg& g = take();
            if (g.kind == AT_END || s_dead) break;
            const uint32_t n = g.n, kfirst = g.k0;
            // this thread's row
            const uint32_t rt = row / a.group, rg = row - rt * a.group;
            const uint32_t tok = g.x * w.tile_tokens + qrow0 + rt;
            const bool real = rt < w.sub_tokens && tok < g.s.nq;
            const int32_t pos = (int32_t)g.s.nkv - (int32_t)g.s.nq + (int32_t)tok;
            int32_t klo = 0, khi = 0x7FFFFFFF;  // a padding row masks nothing: its scores are zeros
            if (real) {
                khi = max(pos + 1, 0);
                klo = a.window ? (int32_t)max((int64_t)pos + 1 - (int64_t)a.window, (int64_t)0) : 0;
            }
            float rs = 1.0f;  // what this row's scores are multiplied by
            bool rescaled = false;
            if constexpr (RESCALE) {
                if (n) {
                    // this row as fp16; by a power of two into its range where its largest is
                    // below 1 or above 2^15: exact down to 2^-24 of the largest
                    at_wait(b_q + 8 * wg, q_phase, &s_dead, err);
                    q_phase ^= 1;
                    const uint32_t base = smb + G::q_off + wg * W * 16384 + row * 128;
                    uint32_t top = 0;
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const uint4 v = at_lds16(base + (i >> 3) * 16384 + ((i ^ row) & 7) * 16);
                        const uint32_t o = max(max(v.x & 0x7F80u, v.y & 0x7F80u), max(v.z & 0x7F80u, v.w & 0x7F80u));
                        const uint32_t h = max(max(v.x & 0x7F800000u, v.y & 0x7F800000u), max(v.z & 0x7F800000u, v.w & 0x7F800000u));
                        top = max(top, max(o, h >> 16));
                    }
                    const uint32_t e = top >> 7;
                    const float f = e < 127 || e > 141 ? at_row_factor(e) : 1.0f;
                    rs = 1.0f / f;
                    rescaled = __any_sync(0xffffffffu, f != 1.0f);
#pragma unroll 4
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t at = base + (i >> 3) * 16384 + ((i ^ row) & 7) * 16;
                        const uint4 v = at_lds16(at);
                        at_sts16(at, make_uint4(at_pack<__half>(bf16_lo(v.x) * f, bf16_hi(v.x) * f),
                                                at_pack<__half>(bf16_lo(v.y) * f, bf16_hi(v.y) * f),
                                                at_pack<__half>(bf16_lo(v.z) * f, bf16_hi(v.z) * f),
                                                at_pack<__half>(bf16_lo(v.w) * f, bf16_hi(v.w) * f)));
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) at_arrive(b_qh + 8 * wg);
                }
            }
            float m = -INFINITY, ref = 0.0f;
            float2 l2[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll 1
            for (uint32_t t = 0; t < n; ++t) {
                const uint32_t buf = NQ == 2 ? wg : (t & 1);
                const uint32_t s_tm = tmem + lanes + buf * 128;
                at_wait(b_s + 8 * buf, s_phase >> buf & 1, &s_dead, err);
                s_phase ^= 1u << buf;
                if (t >= (uint32_t)G::NB) o_phase ^= 1u << buf;
                at_fence_after();
                float s[128];
                {
                    uint32_t* r = reinterpret_cast<uint32_t*>(s);
                    at_ld32(s_tm, r);
                    at_ld32(s_tm + 32, r + 32);
                    at_ld32(s_tm + 64, r + 64);
                    at_ld32(s_tm + 96, r + 96);
                    at_wait_ld();
                }
                const float* sc = reinterpret_cast<const float*>(sm + G::sc_off) + stage * 384;
                if (RESCALE && rescaled) {
#pragma unroll
                    for (int j = 0; j < 128; ++j) s[j] *= rs;
                }
                if constexpr (G::Q8) {
#pragma unroll
                    for (int j = 0; j < 128; j += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(sc + j);
                        const float4 v4 = *reinterpret_cast<const float4*>(sc + 128 + j);
                        const float2 x = at_fma2({s[j], s[j + 1]}, {k4.x, k4.y}, {v4.x, v4.y});
                        const float2 y = at_fma2({s[j + 2], s[j + 3]}, {k4.z, k4.w}, {v4.z, v4.w});
                        s[j] = x.x;
                        s[j + 1] = x.y;
                        s[j + 2] = y.x;
                        s[j + 3] = y.y;
                    }
                }
                const int32_t kt = (int32_t)((kfirst + t) * AT_KEYS);
                if (__any_sync(0xffffffffu, kt < klo || khi - kt < AT_KEYS)) {
                    const uint32_t off = (uint32_t)(kt - klo), span = (uint32_t)(khi > klo ? khi - klo : 0);
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (off + j >= span) s[j] = -INFINITY;
                }
                float mx = fmaxf(s[0], s[1]), mx1 = fmaxf(s[2], s[3]);
#pragma unroll
                for (int j = 4; j < 128; j += 4) {
                    mx = fmaxf(mx, fmaxf(s[j], s[j + 1]));
                    mx1 = fmaxf(mx1, fmaxf(s[j + 2], s[j + 3]));
                }
                mx = fmaxf(mx, mx1);
                if constexpr (!G::Q8) mx *= a.scale_log2;
                const bool up = mx > m + 8.0f || (m == -INFINITY && mx > -INFINITY);
                if (__any_sync(0xffffffffu, up)) {
                    const float f = up ? at_ex2(m - mx) : 1.0f;
                    if (up) m = ref = mx;
                    if (t != 0) {
                        // O so far by the same factor, once the product before this one is in it
                        if (NQ == 1) {
                            at_wait(b_o + 8 * (buf ^ 1), o_phase >> (buf ^ 1) & 1, &s_dead, err);
                            at_fence_after();
                        }
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {  // few at a time: S fills the registers
                            float o[16];
                            at_ld16(o_tm + c, reinterpret_cast<uint32_t*>(o));
                            at_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            at_st16(o_tm + c, reinterpret_cast<uint32_t*>(o));
                        }
                        at_wait_st();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            l2[i].x *= f;
                            l2[i].y *= f;
                        }
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t p[32];
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        float* x = s + half * 64 + j;
                        float2 e0, e1;
                        if constexpr (G::Q8) {
                            e0 = at_add2({x[0], x[1]}, {-ref, -ref});
                            e1 = at_add2({x[2], x[3]}, {-ref, -ref});
                        } else {
                            const float2 k2 = {a.scale_log2, a.scale_log2}, r2 = {-ref, -ref};
                            e0 = at_fma2({x[0], x[1]}, k2, r2);
                            e1 = at_fma2({x[2], x[3]}, k2, r2);
                        }
                        e0 = {at_ex2(e0.x), at_ex2(e0.y)};
                        e1 = {at_ex2(e1.x), at_ex2(e1.y)};
                        if constexpr (G::Q8) {
                            const float4 r4 = *reinterpret_cast<const float4*>(sc + 256 + half * 64 + j);
                            l2[0] = at_fma2(e0, {r4.x, r4.y}, l2[0]);
                            l2[1] = at_fma2(e1, {r4.z, r4.w}, l2[1]);
                        } else {
                            l2[0] = at_add2(l2[0], e0);
                            l2[1] = at_add2(l2[1], e1);
                        }
                        p[j / 2] = at_pack<M>(e0.x, e0.y);
                        p[j / 2 + 1] = at_pack<M>(e1.x, e1.y);
                    }
                    at_st32(s_tm + half * 32, p);
                    at_wait_st();
                    at_fence_before();
                    __syncwarp();
                    if (lane == 0) at_arrive((half ? b_p : b_ph) + 8 * buf);  // a half is multiplied while the other is made
                }
                stage = stage + 1 == NSTAGE ? 0 : stage + 1;
            }
            // ---- the row tile's result ----
            const float l = l2[0].x + l2[0].y + l2[1].x + l2[1].y;
            if (g.n) {
                for (uint32_t t = max(g.n, (uint32_t)G::NB) - G::NB; t < g.n; ++t) take_o(NQ == 2 ? wg : (t & 1));
                at_fence_after();
            }
            const bool bad = (!G::Q8 || ODD8) && *reinterpret_cast<volatile uint32_t*>(&s_bad[seg & 3]) == seg + 1;
            const bool whole = g.kind == AT_FULL;
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;   // l is 0 where the row saw nothing
            const uint32_t slot = 2 * blockIdx.x + (g.kind == AT_FIRST ? 1 : 0);
            unsigned char* part = w.slots + (size_t)slot * w.slot_bytes;
            const uint64_t orow = (uint64_t)(g.s.q0 + tok), ohead = g.h * a.group + rg;
            T* const op = static_cast<T*>(a.out.data) + (int64_t)orow * a.out.ts + (int64_t)ohead * a.out.hs;
            // a lane stores its own row, 32 bytes (a sector) at a time where rows allow it
            const bool wide = ((reinterpret_cast<uintptr_t>(a.out.data) | (uintptr_t)(a.out.ts * 2) | (uintptr_t)(a.out.hs * 2)) & 31) == 0;
            if (bad) {
                // infinities and NaN of v were left out of the products of pieces
                // where not every row sees every key: they go to the rows that do
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    at_ld32(o_tm + c, reinterpret_cast<uint32_t*>(o));
                    at_wait_ld();
                    for (uint32_t t = 0; t < g.n * G::NP; ++t) {
                        const uint32_t key0 = g.k0 * AT_KEYS + t * G::VKEYS;
                        // what was looked over: pieces, and of codes whole tiles
                        if (!real || !at_look(a, g.lo, g.hi, g.p0, ODD8 ? key0 / AT_KEYS * AT_KEYS : key0, ODD8 ? AT_KEYS : G::VKEYS)) continue;
                        const int32_t j0 = max((int32_t)key0, klo);
                        const int32_t j1 = min(min((int32_t)(key0 + G::VKEYS), khi), g.hi);
                        for (int32_t j = j0; j < j1; ++j) {
                            const C* vp;
                            if (a.pages.k) {
                                const int32_t page = ld_now(a.table + (uint64_t)g.b * a.table_width + (j >> a.pages.page_shift));
                                const uint64_t sl = ((uint64_t)(uint32_t)page << a.pages.page_shift) + (j & ((1u << a.pages.page_shift) - 1));
                                if (page < 0 || sl >= a.pages.slots) continue;
                                const uint64_t r = page_row(a.pages, sl, g.h);
                                if (ODD8 && fabsf(a.pages.vs[r]) < CACHE_NOTHING) continue;  // a row of zeros
                                vp = static_cast<const C*>(a.pages.v) + r * D + c;
                            } else {
                                vp = reinterpret_cast<const C*>(static_cast<const T*>(a.v.data) + (int64_t)(g.s.q0 + j) * a.v.ts +
                                                                (int64_t)g.h * a.v.hs + c);
                            }
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                if constexpr (G::Q8) {
                                    if (ODD8 && (reinterpret_cast<const uint8_t*>(vp)[i] & 0x7F) == 0x7F) o[i] = __uint_as_float(0x7FC00000u);
                                } else {
                                    const float v = to_f32(vp[i]);
                                    if (!(fabsf(v) <= 3.4028235e38f)) o[i] += v;
                                }
                            }
                        }
                    }
                    __syncwarp();
                    at_st32(o_tm + c, reinterpret_cast<uint32_t*>(o));
                    at_wait_st();
                }
            }
            // few instructions: they run once a row tile, cold
            if (whole) {
                const float2 inv2 = {inv, inv};
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    if (g.n) {
                        at_ld32(o_tm + c, reinterpret_cast<uint32_t*>(o));
                        at_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = 0.0f;
                    }
                    uint32_t x[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 y = at_mul2({o[2 * i], o[2 * i + 1]}, inv2);
                        x[i] = at_pack<T>(y.x, y.y);
                    }
                    uint4* const p = reinterpret_cast<uint4*>(op + c);
                    if (real && wide) {
                        at_stg32(p, make_uint4(x[0], x[1], x[2], x[3]), make_uint4(x[4], x[5], x[6], x[7]));
                        at_stg32(p + 2, make_uint4(x[8], x[9], x[10], x[11]), make_uint4(x[12], x[13], x[14], x[15]));
                    } else if (real) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                    }
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    at_ld32(o_tm + c, reinterpret_cast<uint32_t*>(o));
                    at_wait_ld();
                    float4* pp = reinterpret_cast<float4*>(part) + (size_t)(c / 4) * G::ROWS + wg * 128 + row;
                    if (real) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) pp[(size_t)(i / 4) * G::ROWS] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
            }
            at_fence_before();
            if (whole) {
                if (a.lse && real)
                    a.lse[orow * a.heads + ohead] = l != 0.0f ? (ref + log2f(l)) * 0.6931471805599453f : -INFINITY;
            } else {
                float2* ml = reinterpret_cast<float2*>(part + (size_t)G::ROWS * D * 4);
                ml[wg * 128 + row] = make_float2(ref, l);
                if (tid == 0) *reinterpret_cast<uint4*>(w.heads + slot * 4) = make_uint4(g.kind, g.b, g.h, g.x);
            }
        }
    } else if (warp < LAST) {
        // ------------------------------ loader ------------------------------
        at_regs_down<G::R_LOAD>();
        const uint32_t lt = (tid - NQ * 128) & 127, lw = (tid - NQ * 128) >> 7;  // lw: which loader warpgroup
        // where 16 bytes c of row r of a piece go: for every 64 dims a block of
        // rows of 128 bytes, swizzled
        auto k_at = [&](uint32_t r, uint32_t c) { return (c >> 3) * (AT_KEYS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
        auto v_at = [&](uint32_t r, uint32_t c) { return (c >> 3) * (G::VKEYS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
        if constexpr (!G::Q8) {
            // 16-bit pieces come by TMA: only V tiles that need a look pass here
            uint32_t before = 0, cleaned = 0;  // pieces of the row tiles before this one, pieces looked over
            for (;; done()) {
                const AtSeg& g = take();
                if (g.kind == AT_END || s_dead) break;
                const int32_t lo = g.lo, hi = g.hi, p0 = g.p0;
                const uint32_t n = g.n, k0 = g.k0;
                for (uint32_t u = 0; u < n * G::NP; ++u) {
                    const uint32_t t = u / G::NP, c = u % G::NP, key0 = (k0 + t) * AT_KEYS + c * G::VKEYS;
                    if (!at_look(a, lo, hi, p0, key0, G::VKEYS)) continue;
                    const uint32_t i = before + (min(n, t + G::LAG) + t) * G::NP + c, slot = i % NSLOT;
                    at_wait(b_raw + 8 * (cleaned % NSLOT), (cleaned / NSLOT) & 1, &s_dead, err);
                    const uint32_t base = smb + G::ring_off + slot * G::PIECE;
                    constexpr uint32_t VU = 8 * W, N = G::PIECE / 2048;
                    const uint32_t r0 = lt / VU, u0 = lt % VU;
                    if ((int32_t)key0 < lo || (int32_t)(key0 + G::VKEYS) > hi) {
#pragma unroll 4
                        for (uint32_t j = 0; j < N; ++j) {
                            const uint32_t r = r0 + j * (128 / VU);
                            const int32_t key = (int32_t)(key0 + r);
                            if (key < lo || key >= hi) at_sts16(base + v_at(r, u0), make_uint4(0, 0, 0, 0));
                        }
                    }
                    uint32_t odd = 0;
#pragma unroll 8
                    for (uint32_t j = 0; j < N; ++j) {
                        const uint4 v = at_lds16(base + v_at(r0 + j * (128 / VU), u0));
                        odd |= at_odd16<T>(v.x) | at_odd16<T>(v.y) | at_odd16<T>(v.z) | at_odd16<T>(v.w);
                    }
                    if (odd & 0x80008000u) {
                        for (uint32_t j = 0; j < N; ++j) {
                            const uint32_t at = base + v_at(r0 + j * (128 / VU), u0);
                            const uint4 v = at_lds16(at);
                            uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const uint32_t m = at_odd16<T>(x[q]);
                                if (m & 0x8000u) x[q] &= 0xFFFF0000u;
                                if (m & 0x80000000u) x[q] &= 0xFFFFu;
                            }
                            at_sts16(at, make_uint4(x[0], x[1], x[2], x[3]));
                        }
                        s_bad[seg & 3] = seg + 1;
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) at_arrive(b_clean + 8 * (cleaned % NSLOT));
                    ++cleaned;
                }
                before += 2 * n * G::NP;
            }
        } else {
            // a warpgroup's 4 x 16 codes a thread are 16 KB of a piece: SUB of them
            // make one, one after the other or by a warpgroup each
            constexpr uint32_t SUB = G::PIECE / 16384 / G::NLD;
            static_assert(G::NLD == 1 || SUB == 1, "loaders");
            uint32_t given = 0, stage = 0;   // parts given to the tensor core
            uint32_t rows_phase = 0;
            // the codes of the two parts issued last (0 older), and what they are: 0 none, 1 K, 2 V
            uint4 raw[2][4];
            uint32_t kind[2] = {0, 0};
            const uint32_t rows0 = smb + G::row_off;
            // thread -> 16 codes: unit u of rows r0, r0 + step, ..; a K part has
            // all rows of 64 dims, a V part 128 / W whole rows
            constexpr uint32_t KU = 4, VU = 4 * W;
            // the older part into its slot, as 16-bit values; the other takes its place
            auto convert = [&]() {
                const uint32_t index = given / SUB, turn = given % SUB, slot = index % NSLOT;
                const uint32_t sub = G::NLD == 2 ? lw : turn;
                const uint32_t base = smb + G::ring_off + slot * G::PIECE;
                if (turn == 0 && index >= (uint32_t)NSLOT) at_wait(b_empty + 8 * slot, (index / NSLOT - 1) & 1, &s_dead, err);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint2 x0 = at_codes(raw[0][i].x, C{}), x1 = at_codes(raw[0][i].y, C{});
                    const uint2 x2 = at_codes(raw[0][i].z, C{}), x3 = at_codes(raw[0][i].w, C{});
                    uint32_t d0, d1;
                    if (kind[0] == 1) {
                        const uint32_t r = lt / KU + i * (128 / KU), c = sub * 8 + 2 * (lt % KU);
                        d0 = k_at(r, c);
                        d1 = k_at(r, c + 1);
                    } else {
                        const uint32_t r = sub * (AT_KEYS / W) + lt / VU + i * (128 / VU), c = 2 * (lt % VU);
                        d0 = v_at(r, c);
                        d1 = v_at(r, c + 1);
                    }
                    at_sts16(base + d0, make_uint4(x0.x, x0.y, x1.x, x1.y));
                    at_sts16(base + d1, make_uint4(x2.x, x2.y, x3.x, x3.y));
                }
                fence_proxy_async();
                __syncwarp();
                if (turn + 1 == SUB && lane == 0) at_arrive(b_full + 8 * slot);
                ++given;
            };
            for (;; done()) {
                const AtSeg& g = take();
                if (g.kind == AT_END || s_dead) break;
                const int32_t lo = g.lo, hi = g.hi;
                const uint32_t n = g.n, k0 = g.k0, head = g.h;
                const int32_t* const table = a.table + (uint64_t)g.b * a.table_width;
                // tiles [calm0, calm1) of V need no look
                const int32_t calm0 = (int32_t)(((int64_t)max((int64_t)lo, a.window ? (int64_t)hi - (int64_t)a.window : 0) + AT_KEYS - 1) >> AT_SHIFT) - (int32_t)k0;
                const int32_t calm1 = (min(hi, g.p0 + 1) >> AT_SHIFT) - (int32_t)k0;
                // part c of a tile of K or V, its rows and scales in stage st
                auto piece = [&](bool is_v, uint32_t c, uint32_t st, bool look) {
                    const uint32_t u = is_v ? lt % VU : lt % KU, r0 = is_v ? lt / VU : lt / KU;
                    const uint32_t step = is_v ? 128 / VU : 128 / KU, key0 = is_v ? c * (AT_KEYS / W) : 0;
                    const uint32_t d = (is_v ? u : c * KU + u) * 16;
                    const C* src = static_cast<const C*>(is_v ? a.pages.v : a.pages.k) + d;
                    uint4 now[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t r = at_lds(rows0 + (st * 2 + (is_v ? 1 : 0)) * 512 + (key0 + r0 + i * step) * 4);
                        now[i] = make_uint4(0, 0, 0, 0);
                        if (r != AT_NONE) now[i] = ld_once(reinterpret_cast<const uint4*>(src + (int64_t)r * D));
                    }
                    if (kind[0]) convert();
                    if (ODD8 && look) {
                        // codes of NaN out of the product: they go to the rows that see them at the end
                        uint32_t odd = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) odd |= at_odd8(now[i].x) | at_odd8(now[i].y) | at_odd8(now[i].z) | at_odd8(now[i].w);
                        if (odd) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                now[i].x &= ~((at_odd8(now[i].x) >> 7) * 0xFFu);
                                now[i].y &= ~((at_odd8(now[i].y) >> 7) * 0xFFu);
                                now[i].z &= ~((at_odd8(now[i].z) >> 7) * 0xFFu);
                                now[i].w &= ~((at_odd8(now[i].w) >> 7) * 0xFFu);
                            }
                            s_bad[seg & 3] = seg + 1;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        raw[0][i] = raw[1][i];
                        raw[1][i] = now[i];
                    }
                    kind[0] = kind[1];
                    kind[1] = is_v ? 2 : 1;
                };
                auto page_of = [&](uint32_t kt) -> int32_t {
                    const int32_t key = (int32_t)(kt * AT_KEYS + lt);
                    return key < lo || key >= hi ? -1 : ld_now(table + (key >> a.pages.page_shift));
                };
                uint32_t kst = stage;
                // A thread a key, each step a tile ahead of the next: its page, then its
                // row's number and scales, then what the others need of them.
                auto row_of = [&](uint32_t kt, int32_t page) -> uint32_t {
                    const int32_t key = (int32_t)(kt * AT_KEYS + lt);
                    if (key < lo || key >= hi) return AT_NONE;
                    const uint64_t slot = ((uint64_t)(uint32_t)page << a.pages.page_shift) +
                                          ((uint32_t)key & ((1u << a.pages.page_shift) - 1));
                    if (page < 0 || slot >= a.pages.slots) {
                        atomicOr(err, SERVE_ERR_PAGE);
                        return AT_NONE;
                    }
                    return (uint32_t)page_row(a.pages, slot, head);
                };
                int32_t page = -1;
                uint32_t r = AT_NONE;
                float ks = 0.0f, vs = 0.0f;
                auto fetch = [&](uint32_t t) {  // row and scales of tile t, page of the one after
                    r = t < n ? row_of(k0 + t, page) : AT_NONE;
                    if (lw == 0 && r != AT_NONE) {
                        ks = a.pages.ks[r];
                        vs = a.pages.vs[r];
                    }
                    if (t + 1 < n) page = page_of(k0 + t + 1);
                };
                if (n) {
                    page = page_of(k0);
                    fetch(0);
                }
                // the row numbers and scales of key tile t into stage kst
                auto resolve = [&](uint32_t t) {
                    if (lw == 0) {
                        // a missing page: scores and values of zero; a scale next to zero: values of zero
                        const bool has = r != AT_NONE, some = has && !(fabsf(vs) < CACHE_NOTHING);
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(rows0 + kst * 1024 + lt * 4), "r"(r) : "memory");
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(rows0 + kst * 1024 + 512 + lt * 4), "r"(some ? r : AT_NONE)
                                     : "memory");
                        float* sc = reinterpret_cast<float*>(sm + G::sc_off) + kst * 384;
                        sc[lt] = has ? ks * a.scale_log2 : 0.0f;
                        sc[128 + lt] = some ? log2f(vs) : 0.0f;
                        // a scale of NaN makes the weights of those who see the key NaN; the others'
                        // weight of 0 must not meet it
                        sc[256 + lt] = !some ? 1.0f : vs == vs ? 1.0f / vs : 0.0f;
                    }
                    // not a barrier of threads: after a failed wait some loaders have left
                    __syncwarp();
                    if (lane == 0) at_arrive(b_rows);
                    at_wait(b_rows, rows_phase, &s_dead, err);
                    rows_phase ^= 1;
                    fetch(t + 1);
                };
                for (uint32_t t = 0; t < (uint32_t)G::LAG && t < n; ++t) {
                    resolve(t);
                    for (uint32_t c = lw; c < (uint32_t)W; c += G::NLD) piece(false, c, kst, false);
                    kst = kst + 1 == NSTAGE ? 0 : kst + 1;
                }
                for (uint32_t t = 0; t < n; ++t) {
                    for (uint32_t c = lw; c < (uint32_t)W; c += G::NLD) piece(true, c, stage, ODD8 && ((int32_t)t < calm0 || (int32_t)t >= calm1));
                    stage = stage + 1 == NSTAGE ? 0 : stage + 1;
                    if (t + G::LAG < n) {
                        resolve(t + G::LAG);
                        for (uint32_t c = lw; c < (uint32_t)W; c += G::NLD) piece(false, c, kst, false);
                        kst = kst + 1 == NSTAGE ? 0 : kst + 1;
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (kind[0]) convert();
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw[0][i] = raw[1][i];
                    kind[0] = kind[1];
                    kind[1] = 0;
                }
            }
        }
    } else {
        at_regs_down<G::R_REST>();
        if (warp == LAST + 1) {
            // ------------------------------ the list of row tiles ------------------------------
            AtWalk walk;
            walk.start(s_plan);
            for (bool more = true; more; ++seg) {
                AtSeg g{};
                more = walk.next(a, w, g);
                if (!more) g.kind = AT_END;
                if (seg >= NSEG) at_wait(b_free + 8 * (seg % NSEG), (seg / NSEG - 1) & 1, &s_dead, err);
                if (s_dead) break;
                if (lane == 0) {
                    small.segs[seg % NSEG] = g;
                    at_arrive(b_seg + 8 * (seg % NSEG));
                }
                __syncwarp();
            }
        } else if (warp == LAST + 2) {
            // ------------------------------ copies ------------------------------
            uint32_t i = 0, raw = 0, last = 0;  // pieces, those to look over; last: parity of a slot's next phase
            uint32_t tiles = 0;                 // row tiles with keys
            const uint32_t ps = a.pages.k ? 1u << a.pages.page_shift : 0;
            const uint32_t nowhere = a.pages.k ? (uint32_t)(a.pages.slots >> a.pages.page_shift) * a.kv_heads : 0;
            for (;; done()) {
                const AtSeg& g = take();
                if (g.kind == AT_END || s_dead) break;
                const int32_t lo = g.lo, hi = g.hi;
                const uint32_t n = g.n, k0 = g.k0, head = g.h, q0 = g.s.q0;
                if (!n) continue;
                // Q: the tile's tokens x the heads of the kv head. Tokens past the
                // sequence are other rows or zeros: padding rows, which nothing reads.
                auto q_tile = [&](uint32_t qi) {
                    if (tiles) at_wait(b_qfree + 8 * qi, (tiles - 1) & 1, &s_dead, err);
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b_q + 8 * qi),
                                     "r"(W * 128 * w.sub_tokens * a.group) : "memory");
                    __syncwarp();
                    if (lane < W)
                        at_tma(smb + G::q_off + (qi * W + lane) * 16384, &qmap, lane * 64, head * a.group,
                               q0 + g.x * w.tile_tokens + qi * w.sub_tokens, b_q + 8 * qi);
                    __syncwarp();
                };
                if constexpr (G::Q8) {
                    for (uint32_t qi = 0; qi < (uint32_t)NQ; ++qi) q_tile(qi);
                    ++tiles;
                    continue;
                }
                const int32_t* const table = a.table + (uint64_t)g.b * a.table_width;
                // keys [key, key + rows) x 64 NB dims from dim d
                auto piece = [&](const CUtensorMap* map, uint32_t key, uint32_t rows, uint32_t d, uint32_t nb, bool look) {
                    const uint32_t slot = i % NSLOT, dst = smb + G::ring_off + slot * G::PIECE;
                    const uint32_t bar = look ? b_raw + 8 * (raw % NSLOT) : b_full + 8 * slot;
                    if (look) ++raw;
                    else last ^= 1u << slot;
                    if (i >= (uint32_t)NSLOT) at_wait(b_empty + 8 * slot, (i / NSLOT - 1) & 1, &s_dead, err);
                    ++i;
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(G::PIECE) : "memory");
                    __syncwarp();
                    const uint32_t box = ps ? min(ps, rows) : rows, per = rows / box;  // boxes a block of 64 dims
                    for (uint32_t j = lane; j < per * nb; j += 32) {
                        const uint32_t blk = j / per, k = key + (j % per) * box;
                        uint32_t y, z;
                        if (ps) {
                            y = k & (ps - 1);
                            z = nowhere;
                            if ((int32_t)(k + box) > lo && (int32_t)k < hi) {
                                const int32_t page = ld_now(table + (k >> a.pages.page_shift));
                                if (page >= 0 && ((uint64_t)(uint32_t)page << a.pages.page_shift) < a.pages.slots)
                                    z = (uint32_t)page * a.kv_heads + head;
                                else
                                    atomicOr(err, SERVE_ERR_PAGE);
                            }
                        } else {
                            y = head * w.head_step;
                            z = q0 + k;
                        }
                        at_tma(dst + blk * (rows * 128) + (j % per) * (box * 128), map, d + blk * 64, y, z, bar);
                    }
                    __syncwarp();
                };
                auto k_tile = [&](uint32_t t) {
                    for (int c = 0; c < G::NP; ++c) piece(&kmap, (k0 + t) * AT_KEYS, AT_KEYS, c * G::KB * 64, G::KB, false);
                };
                q_tile(0);
                k_tile(0);
                if (NQ == 2) q_tile(1);
                ++tiles;
                for (uint32_t t = 1; t < (uint32_t)G::LAG && t < n; ++t) k_tile(t);
                for (uint32_t t = 0; t < n; ++t) {
                    for (int c = 0; c < G::NP; ++c) {
                        const uint32_t key = (k0 + t) * AT_KEYS + c * G::VKEYS;
                        piece(&vmap, key, G::VKEYS, 0, W, at_look(a, lo, hi, g.p0, key, G::VKEYS));
                    }
                    if (t + G::LAG < n) k_tile(t + G::LAG);
                }
            }
            if (s_dead) {
                for (uint32_t j = 0; j < (uint32_t)NQ && tiles; ++j) at_wait_flight(b_q + 8 * j, (tiles - 1) & 1);
                for (uint32_t j = 0; j < (uint32_t)NSLOT && !G::Q8; ++j) {
                    at_wait_flight(b_full + 8 * j, (last >> j & 1) ^ 1);  // true at once for a barrier never used
                    if (raw > j) at_wait_flight(b_raw + 8 * ((raw - 1 - j) % NSLOT), ((raw - 1 - j) / NSLOT) & 1);
                }
            }
        } else if (warp == LAST) {
            // ------------------------------ products ------------------------------
            const uint32_t iqk = at_idesc<M>(AT_KEYS, false), ipv = at_idesc<M>(D, true);
            const uint32_t q0 = smb + G::q_off, ring = smb + G::ring_off;
            // A step multiplies P V of a row tile, then Q K of the tile that its S
            // buffer takes next; the steps of the two row tiles (NQ = 2) or S
            // buffers (NQ = 1) alternate. The whole warp runs the loop, so that
            // addresses and descriptors are uniform, and one lane issues.
            const bool lead = elect_one();
            uint32_t base = 0;            // pieces of the row tiles before this one
            uint32_t cleaned = 0, q_phase = 0, p_phase = 0;
            uint32_t phase = 0;           // bit: parity of the slot's next phase of b_full
            for (;; done()) {
                const AtSeg& g = take();
                if (g.kind == AT_END || s_dead) break;
                const uint32_t n = __shfl_sync(0xffffffffu, g.n, 0);
                if (!n) continue;
                const uint32_t k0 = g.k0;
                const int32_t lo = g.lo, hi = g.hi, p0 = g.p0;
                for (int i = 0; i < NQ; ++i) at_wait((RESCALE ? b_qh : b_q) + 8 * i, q_phase, &s_dead, err);
                q_phase ^= 1;
                const uint32_t steps = NQ == 2 ? 2 * n + 2 : n + 2;
#pragma unroll 1
                for (uint32_t u = 0; u < steps; ++u) {
                    const uint32_t t = NQ == 2 ? u >> 1 : u, qi = NQ == 2 ? u & 1 : 0, buf = u & 1;
                    // with two row tiles a piece is waited for by the first and freed by the second
                    const bool first = NQ == 1 || qi == 0, last = NQ == 1 || qi == 1;
                    if (t >= (uint32_t)G::LAG) {
                        // O += P V of key tile t - LAG; pieces arrive K(0) .. K(LAG - 1), V(0), K(LAG), V(1), ..
                        const uint32_t tv = t - G::LAG;
                        uint32_t slot = (base + (min(n, t) + tv) * G::NP) % NSLOT;
                        at_wait(b_ph + 8 * buf, p_phase >> buf & 1, &s_dead, err);
#pragma unroll
                        for (int c = 0; c < G::NP; ++c) {
                            const bool look = !G::Q8 && first && at_look(a, lo, hi, p0, (k0 + tv) * AT_KEYS + c * G::VKEYS, G::VKEYS);
                            if (look) {
                                at_wait(b_clean + 8 * (cleaned % NSLOT), (cleaned / NSLOT) & 1, &s_dead, err);
                                ++cleaned;
                            } else if (first) {
                                at_wait(b_full + 8 * slot, phase >> slot & 1, &s_dead, err);
                                phase ^= 1u << slot;
                            }
                            const uint32_t bd = at_desc_lo(ring + slot * G::PIECE, G::VKEYS * 128);
                            // P's first 64 keys, then the others (with two pieces: the second)
                            auto pv = [&](int k0, int k1) {
#pragma unroll
                                for (int k = k0; k < k1; ++k)
                                    at_mma_ts(tmem + 256 + qi * D, tmem + buf * 128 + (c * G::VKEYS + k * 16) / 2,
                                              at_desc(bd + k * (2048 >> 4)), ipv, c || k ? 1u : tv);
                            };
                            if (c == 0) {
                                at_fence_after();
                                if (lead) pv(0, 4);
                                __syncwarp();
                            }
                            if (c == G::NP - 1) {
                                at_wait(b_p + 8 * buf, p_phase >> buf & 1, &s_dead, err);
                                p_phase ^= 1u << buf;
                                at_fence_after();
                                if (lead) pv(G::NP == 1 ? 4 : 0, G::VKEYS / 16);
                            }
                            if (lead) {
                                if (last) at_commit(b_empty + 8 * slot);
                                if (c == G::NP - 1) at_commit(b_o + 8 * buf);
                            }
                            __syncwarp();
                            slot = slot + 1 == NSLOT ? 0 : slot + 1;
                        }
                    }
                    if (t < n) {
                        // S = Q K
                        uint32_t slot = (base + (t < (uint32_t)G::LAG ? t : 2 * t - G::LAG + 1) * G::NP) % NSLOT;
#pragma unroll
                        for (int c = 0; c < G::NP; ++c) {
                            if (first) {
                                at_wait(b_full + 8 * slot, phase >> slot & 1, &s_dead, err);
                                phase ^= 1u << slot;
                            }
                            at_fence_after();
                            const uint32_t ad = at_desc_lo(q0 + (qi * W + c * G::KB) * 16384, 16);
                            const uint32_t bd = at_desc_lo(ring + slot * G::PIECE, 16);
                            if (lead) {
#pragma unroll
                                for (int k = 0; k < 4 * G::KB; ++k) {
                                    const uint32_t at = (k >> 2) * (16384 >> 4) + (k & 3) * (32 >> 4);
                                    at_mma_ss(tmem + buf * 128, at_desc(ad + at), at_desc(bd + at), iqk, c || k ? 1u : 0u);
                                }
                                if (last) at_commit(b_empty + 8 * slot);
                                if (c == G::NP - 1) at_commit(b_s + 8 * buf);
                                if (c == G::NP - 1 && t + 1 == n) at_commit(b_qfree + 8 * qi);
                            }
                            __syncwarp();
                            slot = slot + 1 == NSLOT ? 0 : slot + 1;
                        }
                    }
                }
                base += 2 * n * G::NP;
            }
            if (s_dead && lead) {
                at_commit(b_end);
                at_wait_flight(b_end, 0);
            }
        }
        __syncwarp();
    }
    at_fence_before();
    __syncthreads();
    if (warp == LAST) {
        at_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// The row tiles that CTAs share: 32 rows x 64 dims of one tile a CTA, the parts
// added in the order of their keys. blockIdx.x is the CTA that has the tile's
// first keys; blockIdx.y = rows / 32 + dims / 64 * (ROWS / 32).
template <class T, int W, int ROWS>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ ServeAttnArgs a, const __grid_constant__ AtWork w,
                                                        uint32_t ctas) {
    constexpr int D = 64 * W;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = blockIdx.x;
    const uint4 head = ld_once(reinterpret_cast<const uint4*>(w.heads) + 2 * c0 + 1);
    if (head.x != AT_FIRST) return;
    uint32_t parts = 1;
    for (uint32_t j = c0 + 1; j < ctas; j += 32) {
        const uint32_t kind = j + lane < ctas ? ld_once(w.heads + (size_t)(2 * (j + lane)) * 4) : (uint32_t)AT_LAST;
        const uint32_t last = __ballot_sync(0xffffffffu, kind == AT_LAST);
        parts += last ? __ffs(last) : 32;
        if (last) break;
    }
    const uint32_t row = blockIdx.y % (ROWS / 32) * 32 + lane, col = (blockIdx.y / (ROWS / 32) * 8 + warp) * 2;  // float4 pairs
    auto part = [&](uint32_t i) { return w.slots + (size_t)(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * w.slot_bytes; };
    float m = -INFINITY, l = 0.0f;
    float4 o[2] = {};
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < parts; i0 += 4) {
        float2 v[4];
        float4 x[4][2];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            v[i] = make_float2(0.0f, 0.0f);
            if (i0 + i < parts) {
                const float4* p = reinterpret_cast<const float4*>(part(i0 + i)) + (size_t)col * ROWS + row;
                v[i] = ld_once(reinterpret_cast<const float2*>(part(i0 + i) + (size_t)ROWS * D * 4) + row);
                x[i][0] = ld_once(p);
                x[i][1] = ld_once(p + ROWS);
            }
        }
        float top = m;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (v[i].y != 0.0f) top = fmaxf(top, v[i].x);
        const float f0 = l != 0.0f ? at_ex2(m - top) : 0.0f;
        m = top;
        l *= f0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            o[c].x *= f0;
            o[c].y *= f0;
            o[c].z *= f0;
            o[c].w *= f0;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (v[i].y == 0.0f) continue;
            const float f = at_ex2(v[i].x - top);
            l = fmaf(f, v[i].y, l);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                o[c].x = fmaf(f, x[i][c].x, o[c].x);
                o[c].y = fmaf(f, x[i][c].y, o[c].y);
                o[c].z = fmaf(f, x[i][c].z, o[c].z);
                o[c].w = fmaf(f, x[i][c].w, o[c].w);
            }
        }
    }
    const Seq s = seq_of(a, head.y);
    const uint32_t r = row & 127, rt = r / a.group, rg = r - rt * a.group;
    const uint32_t tok = head.w * w.tile_tokens + (row >> 7) * w.sub_tokens + rt;
    if (rt >= w.sub_tokens || tok >= s.nq) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    const uint64_t orow = s.q0 + tok, ohead = head.z * a.group + rg;
    uint4 y;
    y.x = at_pack<T>(o[0].x * inv, o[0].y * inv);
    y.y = at_pack<T>(o[0].z * inv, o[0].w * inv);
    y.z = at_pack<T>(o[1].x * inv, o[1].y * inv);
    y.w = at_pack<T>(o[1].z * inv, o[1].w * inv);
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out.data) + (int64_t)orow * a.out.ts + (int64_t)ohead * a.out.hs + col * 4) = y;
    if (a.lse && col == 0)
        a.lse[orow * a.heads + ohead] = l != 0.0f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace xp
