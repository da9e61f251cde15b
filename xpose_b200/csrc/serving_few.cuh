// Attention of few rows (new tokens x heads of a kv head: 16 at most) over
// pages: the decode step, and the check of a few drafted tokens.
//
// Every key and value is read once and used by all rows, so the time is that
// of reading the cache. The products are warp-wide mma.sync with the keys as
// the long side, S^T = K Q^T and O^T = V^T P^T: 8 * NR rows are its narrow
// side, where the 128-row tiles of tcgen05 would be nearly empty. A warp takes
// 16 or 32 keys at a time from a ring of its own in shared memory, which TMA
// fills by pages in the swizzled layout that ldmatrix reads without conflicts;
// 8-bit codes become exact 16-bit values in registers, and P moves from one
// product's layout to the other's by a transposing register move. Scores of
// 8-bit caches, the running maximum and non-finite values of v are as in the
// tile kernel.
//
// The four warps of a CTA take a step each of a unit of four and add their
// sums in shared memory. CTAs have equal shares of the units of all sequences
// and heads, laid end to end; of a sequence that several share the last to
// finish adds the parts, in their order. (Chunks that CTAs take as they get free
// measured slower: adding the sums of a chunk costs as much as eight units.)
//
// Measured (a call; the device takes the same): 64 sequences of 64 to 16384 keys,
// 32 / 8 heads of 128, e4m3: 80 us, 4.2 TB/s of 342 MB, bound by the instructions
// of 8 warps an SM; one token over 4096 keys, 4 / 1 heads of 256, fp16: 15.5 us, a
// chain of round trips.
#pragma once
#include "serving_tile.cuh"

namespace xp {

template <class T, class C, int W, int NR> struct FwCfg {
    static constexpr int D = 64 * W;
    static constexpr bool Q8 = sizeof(C) == 1;
    static constexpr int RB = D * (int)sizeof(C);            // bytes of a row
    static constexpr int KPS = RB <= 128 ? 32 : 16;          // keys of a warp's step
    static constexpr int UNIT = 4 * KPS;                     // keys of a unit
    static constexpr int SHIFT = KPS == 32 ? 7 : 6;          // log2 UNIT
    static constexpr int HALF = KPS * RB;                    // K of a step, or V
    static constexpr int NST = HALF > 4096 ? (NR == 1 ? 3 : 2) : HALF > 2048 ? 2 : 3;  // steps of a warp's ring
    // two warps' sums at a time, with their m and l; the queries of two items
    static constexpr int ring_bytes = 4 * NST * 2 * HALF;
    static constexpr int scale_off = ring_bytes, scale_bytes = Q8 ? 4 * NST * 2 * KPS * 4 : 0;
    static constexpr int sum_off = scale_off + scale_bytes, sum_bytes = 2 * 8 * NR * (D + 2) * 4;
    static constexpr int q_off = sum_off + sum_bytes, q_bytes = 8 * NR * D * 2;
    static constexpr int smem = q_off + 2 * q_bytes;
    static constexpr int BYTES = smem + 2048;                // with static data and what the system keeps
    static constexpr int CTAS = BYTES > 115000 ? 1 : BYTES > 76000 || W * NR > 4 ? 2 : BYTES > 57000 || W * NR == 4 ? 3 : 4;
};

XP_DEV void fw_cp16(uint32_t dst, const void* src, bool has) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(has ? 16u : 0u) : "memory");
}
XP_DEV void fw_cp4(uint32_t dst, const void* src, bool has) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(has ? 4u : 0u) : "memory");
}
XP_DEV void fw_ldm(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
XP_DEV void fw_ldmt(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
XP_DEV uint32_t fw_movm(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <class T> XP_DEV void fw_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, bf16>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// codes 0 and 2, and 1 and 3, of a word as exact fp16 pairs
XP_DEV uint2 fw_codes_t(uint32_t w, int8c) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4240), b = __byte_perm(u, 0x64646464u, 0x4341);
    const __half2 x = __hsub2(reinterpret_cast<__half2&>(a), bias), y = __hsub2(reinterpret_cast<__half2&>(b), bias);
    return make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
}
XP_DEV uint2 fw_codes_t(uint32_t w, fp8c) { return at_codes(__byte_perm(w, 0, 0x3120), fp8c{}); }
// where 16 bytes c of row r of a step's K or V lie: blocks of 128 bytes of every
// row, in the 128-byte swizzle of the copy (rows of 64 bytes: the 64-byte one),
// so eight rows' equal chunks are in eight bank groups
template <int RB, int KPS> XP_DEV uint32_t fw_at(uint32_t r, uint32_t c) {
    if constexpr (RB >= 128) return (c >> 3) * (KPS * 128) + r * 128 + (((c ^ r) & 7) << 4);
    else return r * 64 + (((c ^ (r >> 1)) & 3) << 4);
}
XP_DEV float fw_lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
XP_DEV float fw_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct FwWork {
    unsigned char* slots;    // partial sums, two of slot_bytes a CTA
    uint32_t* tickets;       // by the CTA with a sequence's first unit: CTAs that are done with it
    uint32_t slot_bytes;
};
constexpr uint32_t FW_COST = 2;  // what a sequence costs besides its units, in units

// The units of all heads and sequences end to end, FW_COST more for each, in
// equal ranges for `ctas` CTAs. Whatever the lengths, the same on every CTA.
struct FwPlan {
    uint64_t total;
    uint32_t ctas;
    uint32_t h, b;           // where this CTA's range starts
    uint32_t skip;           // units of that sequence that earlier CTAs have
    int64_t todo;            // units of the range
};
template <int SHIFT> XP_DEV void fw_make_plan(const ServeAttnArgs& a, uint32_t* sums, FwPlan* out) {
    const uint32_t tid = threadIdx.x;
    uint32_t n = 0, most = 0;
    auto units_of = [&](uint32_t b) -> uint32_t {
        if (b >= a.batch) return 0;
        const Seq s = seq_of(a, b);
        return s.nq ? at_tile(s, 0, 16, a.window, SHIFT).n + FW_COST : 0u;
    };
    uint64_t all = 0;
    uint32_t end = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 128) {
        n = units_of(b0 + tid);
        most = max(most, n);
        uint32_t sum;
        end = at_scan(n, sums, 128, sum);
        all += sum;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if ((tid & 31) == 0) sums[tid >> 5] = most;
    if (tid == 0) out->todo = 0;
    __syncthreads();
    most = max(max(sums[0], sums[1]), max(sums[2], sums[3]));
    __syncthreads();
    // A range of c units takes about c us, adding the n / c parts of a sequence
    // about 1 / 16 us each: c near sqrt(n / 16) is the least of both.
    const uint32_t least = (uint32_t)max(sqrtf((float)most / 16.0f) + 0.5f, 1.0f);
    const uint64_t total = all * a.kv_heads, c = blockIdx.x;
    const uint64_t g = min((uint64_t)gridDim.x, max(at_div(total, least), (uint64_t)1));
    const uint64_t u0 = at_div(total * c, g), u1 = at_div(total * (c + 1), g);
    if (all == 0 || c >= g || u0 == u1) return;
    const uint32_t h = (uint32_t)at_div(u0, all);
    uint64_t at = all * h;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 128) {
        uint32_t sum;
        if (a.batch > 128) {
            n = units_of(b0 + tid);
            end = at_scan(n, sums, 128, sum);
        } else {
            sum = 0;
        }
        const uint64_t e = at + end, s = e - n;
        if (n && s <= u0 && u0 < e) *out = FwPlan{total, (uint32_t)g, h, b0 + tid, (uint32_t)(u0 - s), (int64_t)(u1 - u0)};
        at += sum;
    }
    __syncthreads();
}

// An item as the threads of a CTA see it.
struct FwItem {
    uint32_t h, b, kind;     // head, sequence, AT_FULL .. AT_LAST, or AT_END: no more
    uint32_t k0, n;          // first unit, units
    uint32_t q0, nq;
    uint32_t c0, parts;      // the CTA with the sequence's first unit, CTAs that share it
    int32_t first, lo, hi;   // position of the first new token; the keys that are seen
};

template <class T, class C, int W, int NR>
__global__ void __launch_bounds__(128, (FwCfg<T, C, W, NR>::CTAS))
attn_few_kernel(const __grid_constant__ ServeAttnArgs a, const __grid_constant__ FwWork w,
                const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using G = FwCfg<T, C, W, NR>;
    // 8-bit codes are multiplied in fp16 whatever T is: one conversion makes two
    // of them, and bf16 would need four more operations. bf16 queries enter
    // scaled by a power of two a row (exact down to 2^-24 of the row's largest).
    using M = std::conditional_t<G::Q8, __half, T>;
    constexpr bool RESCALE = G::Q8 && std::is_same_v<T, bf16>;
    constexpr int D = G::D, RB = G::RB, NST = G::NST, KS = D / 16, ROWS = 8 * NR, KPS = G::KPS, KG = KPS / 16;
    constexpr bool Q8 = G::Q8;
    extern __shared__ __align__(1024) unsigned char sm[];
    __shared__ FwPlan s_plan;
    __shared__ uint32_t s_sums[32], s_last;
    __shared__ uint64_t s_bar[4][NST], s_part;
    __shared__ volatile uint32_t s_dead;
    __shared__ FwItem s_desc[2];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lg = lane >> 2, lq = lane & 3;
    const uint32_t ring = smem_u32(sm) + warp * (NST * 2 * G::HALF), qbuf = smem_u32(sm) + G::q_off;
    const uint32_t scales = smem_u32(sm) + G::scale_off + warp * (NST * 2 * KPS * 4), bars = smem_u32(&s_bar[warp][0]);
    if (tid < 4 * NST) {
        mbar_init(&s_bar[0][0] + tid, Q8 ? 33 : 1);  // the copies' lane, and every lane's scales
        fence_mbar_init();
    }
    if (tid == 0) {
        mbar_init(&s_part, 1);
        fence_mbar_init();
        s_dead = 0;
    }
    uint32_t part_phase = 0;
    pdl_launch_dependents();
    pdl_wait();  // everything above may run under the kernel before this one
    fw_make_plan<G::SHIFT>(a, s_sums, &s_plan);
    // The CTA's items. One thread makes them two ahead, so that the ring can
    // run on into the next item while this one's sums are added.
    constexpr uint32_t boss = 96;
    struct {
        uint64_t at;         // where sequence b of head h starts
        uint32_t h, b, skip;
        int64_t todo;
    } walk = {0, 0, 0, 0, 0};
    auto describe = [&]() {
        FwItem x;
        x.kind = AT_END;
        while (walk.todo > 0) {
            const Seq s = seq_of(a, walk.b);
            const AtTile t = at_tile(s, 0, 16, a.window, G::SHIFT);
            const uint32_t all = s.nq ? t.n + FW_COST : 0;
            const uint32_t step = (uint32_t)min((int64_t)(all - walk.skip), walk.todo);
            const uint32_t from = max(walk.skip, FW_COST) - FW_COST, to = max(walk.skip + step, FW_COST) - FW_COST;
            // no unit falls to this CTA: a neighbour has the sequence, or it has none
            const bool some = all && (t.n ? to > from : walk.skip == 0);
            if (some) {
                x.h = walk.h;
                x.b = walk.b;
                x.kind = from == 0 ? (to == t.n ? AT_FULL : AT_FIRST) : (to == t.n ? AT_LAST : AT_MIDDLE);
                x.k0 = t.t0 + from;
                x.n = to - from;
                x.q0 = s.q0;
                x.nq = s.nq;
                x.first = (int32_t)s.nkv - (int32_t)s.nq;
                x.lo = t.lo;
                x.hi = t.hi;
                // the CTAs of the first and last unit: ranges end at floor(total c / ctas)
                const uint64_t total = s_plan.total, g = s_plan.ctas, u0 = walk.at + FW_COST;
                x.c0 = (uint32_t)at_div((u0 + 1) * g + total - 1, total) - 1;
                x.parts = t.n ? (uint32_t)at_div((u0 + t.n) * g + total - 1, total) - x.c0 : 1;
            }
            walk.todo -= step;
            walk.at += all;
            walk.skip = 0;
            if (++walk.b == a.batch) {
                walk.b = 0;
                if (++walk.h == a.kv_heads) walk.todo = 0;
            }
            if (some) break;
        }
        return x;
    };
    if (tid == boss) {
        walk = {0, s_plan.h, s_plan.b, s_plan.skip, s_plan.todo};
        // the range starts `skip` units into its sequence
        if (walk.todo > 0) walk.at = at_div(s_plan.total * blockIdx.x, s_plan.ctas) - walk.skip;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) s_desc[i] = describe();
    }
    __syncthreads();

    // ---- the ring: units of this item, then of the next ----
    uint32_t issued = 0, computed = 0;  // units
    uint32_t phase = 0;                 // bit: parity of the stage's next phase
    uint32_t iu = 0, ipar = 0;          // unit to issue next, in s_desc[ipar]
    bool ahead = false;                 // ... which is the next item
    const uint32_t ps = 1u << a.pages.page_shift, box = min(ps, (uint32_t)KPS);
    const uint32_t nowhere = (uint32_t)(a.pages.slots >> a.pages.page_shift) * a.kv_heads;
    auto step_of = [&](const FwItem& g, uint32_t u) { return (int32_t)((g.k0 + u) * G::UNIT + warp * KPS); };
    auto issue = [&]() {
        const FwItem& g = s_desc[ipar];
        if (iu == 0) {
            // the item's queries, a quarter by each warp: 16-byte pieces, a row's first bits of the piece mixed in
            const uint32_t nrows = g.nq * a.group;
            for (uint32_t id = tid; id < (uint32_t)ROWS * (D / 8); id += 128) {
                const uint32_t r = id / (D / 8), c = id % (D / 8), tok = r / a.group, h = g.h * a.group + (r - tok * a.group);
                const bool has = r < nrows;
                const T* qp = static_cast<const T*>(a.q.data) +
                              (has ? (int64_t)(g.q0 + tok) * a.q.ts + (int64_t)h * a.q.hs + c * 8 : 0);
                fw_cp16(qbuf + ipar * G::q_bytes + r * (D * 2) + ((c ^ (r & 7)) << 4), qp, has);
            }
        }
        const int32_t kb = step_of(g, iu), lo = g.lo, hi = g.hi;
        if (kb < hi && kb + KPS > lo) {
            const uint32_t stage = issued % NST, st = ring + stage * (2 * G::HALF), bar = bars + stage * 8;
            const int32_t* const row = a.table + (uint64_t)g.b * a.table_width;
            if (lane == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * G::HALF) : "memory");
            __syncwarp();
            // a lane a box: pages of the step x blocks of 128 bytes x K and V
            constexpr uint32_t NB = RB >= 128 ? RB / 128 : 1;
            const uint32_t per = KPS / box;
            for (uint32_t j = lane; j < per * NB * 2; j += 32) {
                const uint32_t p = j % per, blk = j / per, kv = blk / NB, nb = blk % NB;
                const int32_t key = kb + (int32_t)(p * box);
                uint32_t z = nowhere;  // past the end: zeros
                if (key < hi && key + (int32_t)box > lo) {
                    const int32_t page = ld_now(row + (key >> a.pages.page_shift));
                    if (page >= 0 && ((uint64_t)(uint32_t)page << a.pages.page_shift) < a.pages.slots)
                        z = (uint32_t)page * a.kv_heads + g.h;
                    else
                        atomicOr(a.err, SERVE_ERR_PAGE);
                }
                at_tma(st + kv * G::HALF + nb * (KPS * 128) + p * box * (RB >= 128 ? 128 : 64), kv ? &vmap : &kmap,
                       nb * (128 / sizeof(C)), (uint32_t)key & (ps - 1), z, bar);
            }
            if constexpr (Q8) {
                const int32_t key = kb + (int32_t)lane;
                bool has = key >= lo && key < hi;
                uint64_t at = 0;
                if (has) {
                    const int32_t page = ld_now(row + (key >> a.pages.page_shift));
                    at = ((uint64_t)(uint32_t)page << a.pages.page_shift) + ((uint32_t)key & (ps - 1));
                    has = page >= 0 && at < a.pages.slots;
                    at = has ? page_row(a.pages, at, g.h) : 0;
                }
                const uint32_t sc = scales + stage * (2 * KPS * 4) + lane * 4;
                if (lane < KPS) {
                    fw_cp4(sc, a.pages.ks + at, has);
                    fw_cp4(sc + KPS * 4, a.pages.vs + at, has);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
            }
        }
        ++iu;
        ++issued;
    };
    // as far as the ring has room and there are units
    auto fill = [&](uint32_t par) {
        while (issued < computed + NST) {
            if (iu >= s_desc[ipar].n) {
                if (ahead || s_desc[par ^ 1].kind == AT_END || s_desc[par ^ 1].n == 0) return;
                ahead = true;
                ipar = par ^ 1;
                iu = 0;
            }
            issue();
        }
    };

    for (uint32_t par = 0; s_desc[par].kind != AT_END; par ^= 1) {
        const FwItem& g = s_desc[par];
        if (!ahead) {
            ipar = par;
            iu = 0;
        }
        ahead = false;
        const uint32_t n = g.n, nrows = g.nq * a.group;
        // rows of this lane: 8 i + lg of Q, 8 i + 2 lq and the next as columns of S^T and O^T
        uint32_t qf[KS][NR][2];
        if (n) {
            fill(par);
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncthreads();  // every warp's part of the queries is in
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const uint32_t r = 8 * i + lg, qr = qbuf + par * G::q_bytes + r * (D * 2);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if constexpr (Q8) {  // the values that stand where the codes of a key's word stand
                        const uint32_t at = qr + (((2 * s + (lq >> 1)) ^ (r & 7)) << 4) + (lq & 1) * 8;
                        qf[s][i][0] = at_lds(at);
                        qf[s][i][1] = at_lds(at + 4);
                    } else {
                        qf[s][i][0] = at_lds(qr + (((2 * s) ^ (r & 7)) << 4) + lq * 4);
                        qf[s][i][1] = at_lds(qr + (((2 * s + 1) ^ (r & 7)) << 4) + lq * 4);
                    }
                }
            }
        }
        float rs[NR][2];  // what a row's scores are multiplied by
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            rs[i][0] = rs[i][1] = a.scale_log2;
            if constexpr (RESCALE) {
                if (n) {
                    uint32_t top = 0;  // the largest exponent of the row
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int j = 0; j < 2; ++j) top = max(top, max(qf[s][i][j] & 0x7F80u, (qf[s][i][j] >> 16) & 0x7F80u));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float f = at_row_factor(top >> 7);
#pragma unroll
                    for (int s = 0; s < KS; ++s)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            qf[s][i][j] = at_pack<__half>(bf16_lo(qf[s][i][j]) * f, bf16_hi(qf[s][i][j]) * f);
#pragma unroll
                    for (int j = 0; j < 2; ++j) rs[i][j] *= 1.0f / __shfl_sync(0xffffffffu, f, (2 * lq + j) * 4);
                }
            }
        }
        int32_t klo[NR][2], khi[NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = 8 * i + 2 * lq + j;
                const int32_t pos = g.first + (int32_t)(r / a.group);
                khi[i][j] = r < nrows ? max(pos + 1, 0) : 0x7FFFFFFF;
                klo[i][j] = r < nrows && a.window ? (int32_t)max((int64_t)pos + 1 - (int64_t)a.window, (int64_t)0) : 0;
            }
        // the keys that every row sees
        int32_t flo = g.lo, fhi = g.hi;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                flo = max(flo, klo[i][j]);
                fhi = min(fhi, khi[i][j]);
            }
        flo = __reduce_max_sync(0xffffffffu, flo);
        fhi = __reduce_min_sync(0xffffffffu, fhi);
        float o[KS][NR][4], m[NR][2], ref[NR][2], l[NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                m[i][j] = -INFINITY;
                ref[i][j] = l[i][j] = 0.0f;
            }
#pragma unroll
            for (int d = 0; d < KS; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[d][i][j] = 0.0f;
        }
        const int32_t lo = g.lo, hi = g.hi;
        const uint32_t k0 = g.k0;
#pragma unroll 1
        for (uint32_t u = 0; u < n; ++u, ++computed) {
            __syncwarp();  // the step before is read: its stage can be filled
            fill(par);
            const int32_t kb = (int32_t)((k0 + u) * G::UNIT + warp * KPS);
            if (kb >= hi || kb + KPS <= lo) continue;
            const uint32_t stage = computed % NST, st = ring + stage * (2 * G::HALF);
            at_wait(bars + stage * 8, phase >> stage & 1, &s_dead, a.err);
            phase ^= 1u << stage;
            const bool partial = kb < flo || kb + KPS > fhi;  // some row does not see some key
            // ---- S^T = K Q^T: blocks of 16 keys ----
            float s[KG][NR][4];
#pragma unroll
            for (int b = 0; b < KG; ++b) {
                float s2[NR][4];
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[b][i][j] = s2[i][j] = 0.0f;
                const uint32_t r = 16 * b + (lane & 15), c0 = lane >> 4;
                if constexpr (Q8) {
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        uint32_t x[4];
                        fw_ldm(st + fw_at<RB, KPS>(r, k + c0), x);
                        const uint2 y0 = at_codes(x[0], C{}), y1 = at_codes(x[1], C{});
                        const uint2 y2 = at_codes(x[2], C{}), y3 = at_codes(x[3], C{});
                        const uint32_t a0[4] = {y0.x, y1.x, y0.y, y1.y}, a1[4] = {y2.x, y3.x, y2.y, y3.y};
#pragma unroll
                        for (int i = 0; i < NR; ++i) {
                            fw_mma<M>(s[b][i], a0, qf[k][i][0], qf[k][i][1]);
                            fw_mma<M>(s2[i], a1, qf[k + 1][i][0], qf[k + 1][i][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        uint32_t x[4];
                        fw_ldm(st + fw_at<RB, KPS>(r, 2 * k + c0), x);
#pragma unroll
                        for (int i = 0; i < NR; ++i) fw_mma<M>(k & 1 ? s2[i] : s[b][i], x, qf[k][i][0], qf[k][i][1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[b][i][j] = (s[b][i][j] + s2[i][j]) * rs[i][j & 1];
            }
            // ---- weights: keys 16 b + lg (values 0, 1) and 8 more (2, 3), rows 2 lq (0, 2) and 2 lq + 1 ----
            float rv[KG][2];
            uint32_t nones = 0;  // 8-bit pages: a bit a key without values
#pragma unroll
            for (int b = 0; b < KG; ++b) rv[b][0] = rv[b][1] = 1.0f;
            if constexpr (Q8) {
                // a lane a key: its scale, log2 of v's and its inverse. Where there is no
                // key or no page (scales of zero), and where v's scale is next to zero, the
                // value is zero: the weight counts with a scale of 1 and multiplies zeros.
                // A scale of NaN makes the weights of those who see the key NaN; the others'
                // weight of 0 must not meet it
                const uint32_t sc = scales + stage * (2 * KPS * 4) + (lane & (KPS - 1)) * 4;
                const float ks0 = __uint_as_float(at_lds(sc)), vs0 = __uint_as_float(at_lds(sc + KPS * 4));
                const bool none = fabsf(vs0) < CACHE_NOTHING;
                nones = __ballot_sync(0xffffffffu, none);
                const float lv0 = none ? 0.0f : fw_lg2(vs0);
                const float rv0 = none ? 1.0f : vs0 == vs0 ? fw_rcp(vs0 * 0x1p-10f) * 0x1p-10f : 0.0f;  // may be subnormal
#pragma unroll
                for (int b = 0; b < KG; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t from = 16 * b + 8 * h + lg;
                        const float ks = __shfl_sync(0xffffffffu, ks0, from), lv = __shfl_sync(0xffffffffu, lv0, from);
                        rv[b][h] = __shfl_sync(0xffffffffu, rv0, from);
#pragma unroll
                        for (int i = 0; i < NR; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) s[b][i][2 * h + j] = fmaf(s[b][i][2 * h + j], ks, lv);
                    }
            }
            if (partial) {
#pragma unroll
                for (int b = 0; b < KG; ++b)
#pragma unroll
                    for (int i = 0; i < NR; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int32_t key = kb + 16 * b + (int32_t)lg + 8 * (j >> 1);
                            if (key < klo[i][j & 1] || key >= khi[i][j & 1] || key >= hi || key < lo) s[b][i][j] = -INFINITY;
                        }
            }
            bool up = false;
#pragma unroll
            for (int b = 0; b < KG; ++b)
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) up |= s[b][i][j] > m[i][j & 1] + 8.0f;
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = fmaxf(s[0][i][j], s[0][i][j + 2]);
#pragma unroll
                        for (int b = 1; b < KG; ++b) x = fmaxf(x, fmaxf(s[b][i][j], s[b][i][j + 2]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        if (x > m[i][j]) {
                            const float f = at_ex2(m[i][j] - x);
                            m[i][j] = ref[i][j] = x;
                            l[i][j] *= f;
#pragma unroll
                            for (int d = 0; d < KS; ++d) {
                                o[d][i][j] *= f;
                                o[d][i][j + 2] *= f;
                            }
                        }
                    }
            }
            uint32_t pb[KG][NR][2];
#pragma unroll
            for (int b = 0; b < KG; ++b)
#pragma unroll
                for (int i = 0; i < NR; ++i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[b][i][j] = at_ex2(s[b][i][j] - ref[i][j & 1]);
                        l[i][j & 1] = fmaf(s[b][i][j], rv[b][j >> 1], l[i][j & 1]);
                    }
                    pb[b][i][0] = fw_movm(at_pack<M>(s[b][i][0], s[b][i][1]));
                    pb[b][i][1] = fw_movm(at_pack<M>(s[b][i][2], s[b][i][3]));
                }
            // ---- O^T += V^T P^T ----
            const uint32_t sv = st + G::HALF;
            if constexpr (std::is_same_v<C, fp8c>) {
                // where some row does not see what another sees: codes of NaN only to the rows
                // that see them, out of the step's V and into their sums
                if ((kb < flo && lo < flo) || (kb + KPS > fhi && fhi < hi)) {
                    uint32_t odd = 0;
#pragma unroll 1
                    for (uint32_t c = lane * 16; c < (uint32_t)G::HALF; c += 512) {
                        const uint4 v = at_lds16(sv + c);
                        odd |= at_odd8(v.x) | at_odd8(v.y) | at_odd8(v.z) | at_odd8(v.w);
                    }
                    if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
                        for (int d = 0; d < KS; ++d)
                            for (uint32_t j = 0; j < (uint32_t)KPS; ++j) {
                                if (nones >> j & 1) continue;
                                const int32_t key = kb + (int32_t)j;
                                // the lane's two dims
                                uint16_t two;
                                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(two) : "r"(sv + fw_at<RB, KPS>(j, d) + lg * 2) : "memory");
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    if ((two >> (8 * half) & 0x7F) != 0x7F) continue;
#pragma unroll
                                    for (int i = 0; i < NR; ++i)
#pragma unroll
                                        for (int q = 0; q < 2; ++q)
                                            if (key >= klo[i][q] && key < khi[i][q])
                                                o[d][i][2 * half + q] = __uint_as_float(0x7FC00000u);
                                }
                            }
                        __syncwarp();
#pragma unroll 1
                        for (uint32_t c = lane * 16; c < (uint32_t)G::HALF; c += 512) {
                            uint4 v = at_lds16(sv + c);
                            v.x &= ~((at_odd8(v.x) >> 7) * 0xFFu);
                            v.y &= ~((at_odd8(v.y) >> 7) * 0xFFu);
                            v.z &= ~((at_odd8(v.z) >> 7) * 0xFFu);
                            v.w &= ~((at_odd8(v.w) >> 7) * 0xFFu);
                            at_sts16(sv + c, v);
                        }
                        fence_proxy_async();  // before the next copy over them
                        __syncwarp();
                    }
                }
            }
            if constexpr (Q8) {
                const uint32_t r = lane & 15, c0 = lane >> 4;
#pragma unroll
                for (int b = 0; b < KG; ++b) {
                    // rows without values, and those that are no keys, may hold anything, codes of NaN among it
                    uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (nones) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t two = nones >> (16 * b + 8 * h + 2 * lq);
                            keep[h] = (two & 1 ? 0u : 0xFFFFu) | (two & 2 ? 0u : 0xFFFF0000u);
                        }
                    }
#pragma unroll
                    for (int d = 0; d < KS; d += 2) {
                        uint32_t x[4];
                        fw_ldmt(sv + fw_at<RB, KPS>(16 * b + r, d + c0), x);
                        if (nones) {
                            x[0] &= keep[0];
                            x[1] &= keep[1];
                            x[2] &= keep[0];
                            x[3] &= keep[1];
                        }
                        // a dim's two keys side by side
                        const uint2 y0 = fw_codes_t(x[0], C{}), y1 = fw_codes_t(x[1], C{});
                        const uint2 y2 = fw_codes_t(x[2], C{}), y3 = fw_codes_t(x[3], C{});
                        const uint32_t a0[4] = {y0.x, y0.y, y1.x, y1.y}, a1[4] = {y2.x, y2.y, y3.x, y3.y};
#pragma unroll
                        for (int i = 0; i < NR; ++i) {
                            fw_mma<M>(o[d][i], a0, pb[b][i][0], pb[b][i][1]);
                            fw_mma<M>(o[d + 1][i], a1, pb[b][i][0], pb[b][i][1]);
                        }
                    }
                }
            } else {
                const uint32_t r = (lane & 7) + (lane >> 4) * 8, c0 = (lane >> 3) & 1;
                constexpr uint32_t mask = std::is_same_v<T, bf16> ? 0x7F80u : 0x7C00u;
                bool odd = false;
#pragma unroll
                for (int b = 0; b < KG; ++b)
#pragma unroll
                    for (int d = 0; d < KS; ++d) {
                        uint32_t x[4];
                        fw_ldmt(sv + fw_at<RB, KPS>(16 * b + r, 2 * d + c0), x);
                        if (partial) {  // infinities and NaN only to the rows that see them
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int32_t key = kb + 16 * b + 8 * (j >> 1) + 2 * (int32_t)lq;
                                if (key < lo || key >= hi) x[j] &= 0xFFFF0000u;
                                if (key + 1 < lo || key + 1 >= hi) x[j] &= 0xFFFFu;
                                if ((x[j] & mask) == mask) { x[j] &= 0xFFFF0000u; odd = true; }
                                if ((x[j] & (mask << 16)) == (mask << 16)) { x[j] &= 0xFFFFu; odd = true; }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < NR; ++i) fw_mma<M>(o[d][i], x, pb[b][i][0], pb[b][i][1]);
                    }
                if (partial && __any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int d = 0; d < KS; ++d)
                        for (uint32_t j = 0; j < (uint32_t)KPS; ++j) {
                            const int32_t key = kb + (int32_t)j;
                            if (key < lo || key >= hi) continue;
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                T v;
                                asm volatile("ld.shared.u16 %0, [%1];"
                                             : "=h"(reinterpret_cast<uint16_t&>(v))
                                             : "r"(sv + fw_at<RB, KPS>(j, 2 * d + half) + lg * 2)
                                             : "memory");
                                const float x = to_f32(v);
                                if (fabsf(x) <= 3.4028235e38f) continue;
#pragma unroll
                                for (int i = 0; i < NR; ++i)
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        if (key >= klo[i][q] && key < khi[i][q]) o[d][i][2 * half + q] += x;
                            }
                        }
                }
            }
        }
        // ---- the warps' sums: 2 and 3 to 0 and 1, those two to all ----
        float* const so = reinterpret_cast<float*>(sm + G::sum_off);                     // [2][ROWS][D]
        float2* const sml = reinterpret_cast<float2*>(sm + G::sum_off + 2 * ROWS * D * 4);  // [2][ROWS] m, l
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], d);
        // value k of a lane's four dims, two rows
        auto at_o = [&](uint32_t r, int d, int half) {
            return so + ((warp & 1) * ROWS + r) * D + d * 16 + (Q8 ? 2 * lg + half : lg + 8 * half);
        };
        auto put = [&]() {
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t r = 8 * i + 2 * lq + j;
                    if (r >= nrows) continue;
                    if (lg == 0) sml[(warp & 1) * ROWS + r] = make_float2(ref[i][j], l[i][j]);
#pragma unroll
                    for (int d = 0; d < KS; ++d) {
                        *at_o(r, d, 0) = o[d][i][j];
                        *at_o(r, d, 1) = o[d][i][j + 2];
                    }
                }
        };
        __syncthreads();  // the sums of the item before are read
        if (warp >= 2) put();
        __syncthreads();
        if (warp < 2) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t r = 8 * i + 2 * lq + j;
                    if (r >= nrows) continue;
                    const float2 v = sml[warp * ROWS + r];
                    // a side without weight (l = 0) has no say in the maximum
                    const float m0 = l[i][j] != 0.0f ? ref[i][j] : -INFINITY, m1 = v.y != 0.0f ? v.x : -INFINITY;
                    const float top = fmaxf(m0, m1);
                    const float f0 = l[i][j] != 0.0f ? at_ex2(m0 - top) : 0.0f, f1 = v.y != 0.0f ? at_ex2(m1 - top) : 0.0f;
                    ref[i][j] = l[i][j] != 0.0f || v.y != 0.0f ? top : 0.0f;
                    l[i][j] = l[i][j] * f0 + v.y * f1;
#pragma unroll
                    for (int d = 0; d < KS; ++d) {
                        o[d][i][j] = o[d][i][j] * f0 + *at_o(r, d, 0) * f1;
                        o[d][i][j + 2] = o[d][i][j + 2] * f0 + *at_o(r, d, 1) * f1;
                    }
                }
            __syncwarp();
            put();
        }
        __syncthreads();
        const bool whole = g.kind == AT_FULL;
        unsigned char* const part = w.slots + (size_t)(2 * blockIdx.x + (g.kind == AT_FIRST)) * w.slot_bytes;
        auto emit = [&](uint32_t r, uint32_t c, float4 x, float mm, float ll) {
            const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
            const uint32_t tok = r / a.group, h = g.h * a.group + (r - tok * a.group);
            uint2 y;
            y.x = at_pack<T>(x.x * inv, x.y * inv);
            y.y = at_pack<T>(x.z * inv, x.w * inv);
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out.data) + (int64_t)(g.q0 + tok) * a.out.ts + (int64_t)h * a.out.hs +
                                      4 * c) = y;
            if (a.lse && c == 0)
                a.lse[(uint64_t)(g.q0 + tok) * a.heads + h] = ll != 0.0f ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
        };
        for (uint32_t id = tid; id < nrows * (D / 4); id += 128) {
            const uint32_t r = id / (D / 4), c = id % (D / 4);
            const float2 v0 = sml[r], v1 = sml[ROWS + r];
            const float m0 = v0.y != 0.0f ? v0.x : -INFINITY, m1 = v1.y != 0.0f ? v1.x : -INFINITY, top = fmaxf(m0, m1);
            const float f0 = v0.y != 0.0f ? at_ex2(m0 - top) : 0.0f, f1 = v1.y != 0.0f ? at_ex2(m1 - top) : 0.0f;
            const float4 y0 = *reinterpret_cast<const float4*>(so + r * D + 4 * c);
            const float4 y1 = *reinterpret_cast<const float4*>(so + (ROWS + r) * D + 4 * c);
            const float ll = v0.y * f0 + v1.y * f1;
            const float4 x = make_float4(y0.x * f0 + y1.x * f1, y0.y * f0 + y1.y * f1, y0.z * f0 + y1.z * f1, y0.w * f0 + y1.w * f1);
            if (whole) {
                emit(r, c, x, top, ll);
            } else {
                __stcg(reinterpret_cast<float4*>(part + ROWS * 8) + id, x);
                if (c == 0) __stcg(reinterpret_cast<float2*>(part) + r, make_float2(ll != 0.0f ? top : 0.0f, ll));
            }
        }
        if (!whole) {
            const uint32_t c0 = g.c0, nparts = g.parts;
            constexpr uint32_t PER = (ROWS * (D / 4) + 127) / 128;  // float4 of a thread
            fence_proxy_async_all();  // the last CTA reads the parts by bulk copies
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = atomicAdd(w.tickets + c0, 1u) == nparts - 1;
                if (s_last) w.tickets[c0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                // The parts (m and l of every row, then the sums) come into shared
                // memory by bulk copies: the ring, if no next item runs on in it,
                // else the small buffer of the sums. Little code, because it runs
                // once: what is not in the instruction cache costs more than it does.
                const bool idle = s_desc[par ^ 1].kind == AT_END;
                unsigned char* const buf = sm + (idle ? 0 : G::sum_off);
                const uint32_t bytes = ROWS * 8 + nrows * (D * 4);
                const uint32_t fit = (idle ? (uint32_t)G::ring_bytes : (uint32_t)G::sum_bytes) / bytes;
                float4 x[PER];
                float mm[PER], ll[PER];
#pragma unroll
                for (uint32_t k = 0; k < PER; ++k) {
                    x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    mm[k] = -INFINITY;
                    ll[k] = 0.0f;
                }
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < nparts; i0 += fit) {
                    const uint32_t m = min(nparts - i0, fit);
                    __syncthreads();
                    // what other CTAs wrote as parts before the copies read it, and what
                    // the threads wrote in the buffer before the copies write there
                    fence_proxy_async_all();
                    if (tid == 0)
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&s_part)),
                                     "r"(m * bytes) : "memory");
                    __syncthreads();
                    for (uint32_t i = tid; i < m; i += 128) {
                        const uint32_t p = i0 + i;
                        bulk_g2s(buf + i * bytes, w.slots + (size_t)(p ? 2 * (c0 + p) : 2 * c0 + 1) * w.slot_bytes, bytes, &s_part);
                    }
                    at_wait(smem_u32(&s_part), part_phase, &s_dead, a.err);
                    part_phase ^= 1;
#pragma unroll
                    for (uint32_t k = 0; k < PER; ++k) {
                        const uint32_t id = tid + k * 128, r = id / (D / 4);
                        if (r >= nrows) break;
                        float top = mm[k];
#pragma unroll 4
                        for (uint32_t i = 0; i < m; ++i) {
                            const float2 v = *reinterpret_cast<const float2*>(buf + i * bytes + r * 8);
                            top = fmaxf(top, v.y != 0.0f ? v.x : -INFINITY);
                        }
                        const float f0 = ll[k] != 0.0f ? at_ex2(mm[k] - top) : 0.0f;
                        mm[k] = top;
                        ll[k] *= f0;
                        x[k].x *= f0;
                        x[k].y *= f0;
                        x[k].z *= f0;
                        x[k].w *= f0;
#pragma unroll 4
                        for (uint32_t i = 0; i < m; ++i) {
                            const float2 v = *reinterpret_cast<const float2*>(buf + i * bytes + r * 8);
                            const float4 y = *reinterpret_cast<const float4*>(buf + i * bytes + ROWS * 8 + id * 16);
                            const float f = v.y != 0.0f ? at_ex2(v.x - top) : 0.0f;
                            ll[k] = fmaf(f, v.y, ll[k]);
                            x[k].x = fmaf(f, y.x, x[k].x);
                            x[k].y = fmaf(f, y.y, x[k].y);
                            x[k].z = fmaf(f, y.z, x[k].z);
                            x[k].w = fmaf(f, y.w, x[k].w);
                        }
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < PER; ++k) {
                    const uint32_t id = tid + k * 128, r = id / (D / 4);
                    if (r < nrows) emit(r, id % (D / 4), x[k], mm[k], ll[k]);
                }
            }
        }
        __syncthreads();  // nobody needs s_desc[par] any more
        if (tid == boss) s_desc[par] = describe();
        __syncthreads();
    }
    if (s_dead) {  // copies may still be on their way into this CTA's memory
        __syncthreads();
        if (tid < 4 * NST)
            for (int i = 0; i < 2; ++i) at_wait_flight(smem_u32(&s_bar[0][0] + tid), i);
        __syncthreads();
    }
    at_clear<T, D>(a, 128);
}

}  // namespace xp
