// Attention of few rows (new tokens x heads of a kv head: 16 at most) over
// pages: the decode step, and the check of a few drafted tokens.
//
// Every key and value is read once and used by all rows, so the time is that
// of reading the cache. The products are warp-wide mma.sync with the keys as
// the long side, S^T = K Q^T and O^T = V^T P^T: 8 * NR rows are its narrow
// side, where the 128-row tiles of tcgen05 would be nearly empty. A warp takes
// 16 keys at a time from a ring of its own in shared memory (cp.async; keys
// outside the range are zeros), 8-bit codes become exact 16-bit values in
// registers, and P moves from one product's layout to the other's by a
// transposing register move. Scores of 8-bit caches, the running maximum and
// non-finite values of v are as in the tile kernel.
//
// The four warps of a CTA take 16 keys each of a unit of 64 and add their sums
// in shared memory. Long sequences are cut into chunks of units, about four
// for every CTA on the GPU, which the CTAs take as they get free: SMs do not
// read at the same speed, and equal shares left the slow ones a fifth behind.
// The last CTA of a sequence to finish adds its chunks, in their order.
#pragma once
#include "serving_tile.cuh"

namespace xp {

template <class T, class C, int W, int NR> struct FwCfg {
    static constexpr int D = 64 * W;
    static constexpr bool Q8 = sizeof(C) == 1;
    static constexpr int RB = D * (int)sizeof(C);            // bytes of a row
    static constexpr int STAGE = 2 * 16 * RB + (Q8 ? 128 : 0);  // 16 keys: K, V, scales
    static constexpr int NST = STAGE > 4100 ? 2 : STAGE > 2200 ? 3 : 4;  // stages of a warp's ring
    // two warps' sums at a time, with their m and l; the queries of two items
    static constexpr int ring_bytes = 4 * NST * STAGE;
    static constexpr int sum_off = ring_bytes, sum_bytes = 2 * 8 * NR * (D + 2) * 4;
    static constexpr int q_off = sum_off + sum_bytes, q_bytes = 8 * NR * D * 2;
    static constexpr int ends_off = q_off + 2 * q_bytes;     // a word a sequence
    static constexpr int BYTES = ends_off + 1024;            // ... of 128 sequences, and static
    static constexpr int CTAS = BYTES > 115000 ? 1 : BYTES > 76000 || W * NR > 4 ? 2 : BYTES > 57500 || W * NR == 4 ? 3 : 4;
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
XP_DEV uint2 fw_codes_t(uint32_t w, fp8c) { return at_codes<__half>(__byte_perm(w, 0, 0x3120), fp8c{}); }
// where 16 bytes c of row r of a stage lie: eight rows' equal chunks in eight bank groups
template <int RB> XP_DEV uint32_t fw_at(uint32_t r, uint32_t c) {
    if constexpr (RB >= 128) return r * RB + ((c & ~7u) << 4) + (((c ^ r) & 7) << 4);
    else return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (r >> 1)) & 7) * 16;
}

struct FwWork {
    unsigned char* slots;    // partial sums of the chunks of split sequences, by item
    uint32_t* tickets;       // by item: chunks of the sequence that starts there that are done
    uint32_t* counters;      // [0] items taken beyond the first of every CTA, [1] CTAs that ended
    uint32_t slot_bytes, most_slots;
};

// An item: chunk c of n of head h of sequence b; items are numbered by head,
// sequence, chunk. Whatever the lengths, the same on every CTA.
struct FwPlan {
    uint32_t per_head, chunk;  // items a head, units a chunk
};
// `ends`: a word a sequence, where its items end. A sequence without new
// tokens has none; one without keys has one.
XP_DEV FwPlan fw_make_plan(const ServeAttnArgs& a, const FwWork& w, uint32_t* ends, uint32_t* sums) {
    const uint32_t tid = threadIdx.x;
    uint32_t n = 0;
    auto units_of = [&](uint32_t b) -> uint32_t {  // 0: no items
        if (b >= a.batch) return 0;
        const Seq s = seq_of(a, b);
        return s.nq ? max(at_tile(s, 0, 16, a.window, 6).n, 1u) : 0u;
    };
    uint64_t all = 0;
    uint32_t most = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 128) {
        n = units_of(b0 + tid);
        most = max(most, n);
        uint32_t sum;
        at_scan(n, sums, 128, sum);
        all += sum;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if ((tid & 31) == 0) sums[tid >> 5] = most;
    __syncthreads();
    most = max(max(sums[0], sums[1]), max(sums[2], sums[3]));
    // One chunk a CTA while there are at most a few units for each, else four.
    // A chunk of c units takes about c / 2 us, adding the n / c chunks of a
    // sequence about 1 / 24 us each: c near sqrt(n / 12) is the least of both.
    all *= a.kv_heads;
    const uint64_t ctas = gridDim.x;
    uint64_t chunk = all <= 8 * ctas ? (all + ctas - 1) / ctas : (all + 4 * ctas - 1) / (4 * ctas);
    chunk = max(chunk, (uint64_t)max(sqrtf((float)most / 12.0f) + 0.5f, 1.0f));
    FwPlan p;
    for (;;) {
        p.chunk = (uint32_t)min(chunk, (uint64_t)0x7FFFFFFF);
        uint32_t items = 0;
        for (uint32_t b0 = 0; b0 < a.batch; b0 += 128) {
            if (a.batch > 128) n = units_of(b0 + tid);
            uint32_t sum;
            const uint32_t end = items + at_scan(n ? (n - 1) / p.chunk + 1 : 0, sums, 128, sum);
            if (b0 + tid < a.batch) ends[b0 + tid] = end;
            items += sum;
        }
        p.per_head = items;
        // more items than partial sums have room for: so many sequences need no cut
        if ((uint64_t)items * a.kv_heads <= w.most_slots || p.chunk == 0x7FFFFFFF) break;
        chunk = 0x7FFFFFFF;
        __syncthreads();
    }
    __syncthreads();
    return p;
}

// An item as the threads of a CTA see it.
struct FwItem {
    uint32_t h, b, ch, nch;  // head, sequence, chunk and of how many
    uint32_t k0, n;          // first unit, units
    uint32_t q0, nq;
    int32_t first, lo, hi;   // position of the first new token; the keys that are seen
};

template <class T, class C, int W, int NR>
__global__ void __launch_bounds__(128, (FwCfg<T, C, W, NR>::CTAS))
attn_few_kernel(const __grid_constant__ ServeAttnArgs a, const __grid_constant__ FwWork w) {
    using G = FwCfg<T, C, W, NR>;
    // 8-bit codes are multiplied in fp16 whatever T is: one conversion makes two
    // of them, and bf16 would need four more operations. bf16 queries enter
    // scaled by a power of two a row (exact down to 2^-24 of the row's largest).
    using M = std::conditional_t<G::Q8, __half, T>;
    constexpr bool RESCALE = G::Q8 && std::is_same_v<T, bf16>;
    constexpr int D = G::D, RB = G::RB, NST = G::NST, KS = D / 16, ROWS = 8 * NR;
    constexpr bool Q8 = G::Q8;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ uint32_t s_sums[32], s_last, s_item[2];
    __shared__ FwItem s_desc[2];
    uint32_t* const ends = reinterpret_cast<uint32_t*>(sm + G::ends_off);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lg = lane >> 2, lq = lane & 3;
    const uint32_t ring = smem_u32(sm) + warp * (NST * G::STAGE), qbuf = smem_u32(sm) + G::q_off;
    const FwPlan plan = fw_make_plan(a, w, ends, s_sums);
    const uint32_t items = plan.per_head * a.kv_heads;
    auto describe = [&](uint32_t item) {
        FwItem x;
        x.h = item / plan.per_head;
        const uint32_t i = item - x.h * plan.per_head;
        uint32_t lo = 0, hi = a.batch - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (ends[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        x.b = lo;
        const uint32_t begin = lo ? ends[lo - 1] : 0;
        x.nch = ends[lo] - begin;
        x.ch = i - begin;
        const Seq s = seq_of(a, x.b);
        const AtTile t = at_tile(s, 0, 16, a.window, 6);
        x.q0 = s.q0;
        x.nq = s.nq;
        x.first = (int32_t)s.nkv - (int32_t)s.nq;
        x.lo = t.lo;
        x.hi = t.hi;
        x.k0 = t.t0 + x.ch * plan.chunk;
        x.n = t.n ? min(plan.chunk, t.n - x.ch * plan.chunk) : 0;
        return x;
    };
    // The CTA's items: the first by its number, the others from a counter. One
    // thread fetches them two ahead, so that the ring can run on into the next
    // item while this one's sums are added.
    const uint32_t boss = 96;
    uint32_t fetched = 0;
    if (tid == boss) {
        s_item[0] = blockIdx.x;
        s_item[1] = blockIdx.x < items ? gridDim.x + atomicAdd(w.counters, 1u) : items;
        for (int i = 0; i < 2; ++i)
            if (s_item[i] < items) s_desc[i] = describe(s_item[i]);
    }
    __syncthreads();

    // ---- the ring: units of this item, then of the next ----
    uint32_t issued = 0, computed = 0;  // units
    uint32_t iu = 0, ipar = 0;          // unit to issue next, in s_desc[ipar]
    bool ahead = false;                 // ... which is the next item
    int32_t page = -1;
    auto page_of = [&](const FwItem& g, uint32_t u) -> int32_t {  // lane & 15: the key
        const int32_t key = (int32_t)((g.k0 + u) * 64 + warp * 16 + (lane & 15));
        return u < g.n && key >= g.lo && key < g.hi
                   ? __ldg(a.table + (uint64_t)g.b * a.table_width + (key >> a.pages.page_shift))
                   : -1;
    };
    auto issue = [&]() {
        const FwItem& g = s_desc[ipar];
        if (iu == 0) {
            // the item's queries, a quarter by each warp: 16-byte pieces, a row's first bits of the piece mixed in
            page = page_of(g, 0);
            const uint32_t nrows = g.nq * a.group;
            for (uint32_t id = tid; id < (uint32_t)ROWS * (D / 8); id += 128) {
                const uint32_t r = id / (D / 8), c = id % (D / 8), tok = r / a.group, h = g.h * a.group + (r - tok * a.group);
                const bool has = r < nrows;
                const T* qp = static_cast<const T*>(a.q.data) +
                              (has ? (int64_t)(g.q0 + tok) * a.q.ts + (int64_t)h * a.q.hs + c * 8 : 0);
                fw_cp16(qbuf + ipar * G::q_bytes + r * (D * 2) + ((c ^ (r & 7)) << 4), qp, has);
            }
        }
        const int32_t kb = (int32_t)((g.k0 + iu) * 64 + warp * 16);
        if (kb < g.hi && kb + 16 > g.lo) {
            const int32_t key = kb + (int32_t)(lane & 15);
            uint32_t row = AT_NONE;
            if (key >= g.lo && key < g.hi) {
                const uint64_t slot = ((uint64_t)(uint32_t)page << a.pages.page_shift) +
                                      ((uint32_t)key & ((1u << a.pages.page_shift) - 1));
                if (page < 0 || slot >= a.pages.slots) atomicOr(a.err, SERVE_ERR_PAGE);
                else row = (uint32_t)page_row(a.pages, slot, g.h);
            }
            const uint32_t st = ring + (issued % NST) * G::STAGE;
            constexpr uint32_t PR = RB / 16;
#pragma unroll
            for (uint32_t i = 0; i < PR / 2; ++i) {
                const uint32_t id = i * 32 + lane, r = id / PR, c = id % PR;
                const uint32_t x = __shfl_sync(0xffffffffu, row, r);
                const bool has = x != AT_NONE;
                const uint64_t off = has ? (uint64_t)x * RB + c * 16 : 0;
                fw_cp16(st + fw_at<RB>(r, c), static_cast<const char*>(a.pages.k) + off, has);
                fw_cp16(st + 16 * RB + fw_at<RB>(r, c), static_cast<const char*>(a.pages.v) + off, has);
            }
            if constexpr (Q8) {
                const bool has = row != AT_NONE;
                fw_cp4(st + 32 * RB + lane * 4, (lane < 16 ? a.pages.ks : a.pages.vs) + (has ? row : 0), has);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        page = page_of(g, ++iu);
        ++issued;
    };
    // as far as the ring has room and there are units
    auto fill = [&](uint32_t par) {
        while (issued < computed + NST) {
            if (iu >= s_desc[ipar].n) {
                if (ahead || s_item[par ^ 1] >= items || s_desc[par ^ 1].n == 0) return;
                ahead = true;
                ipar = par ^ 1;
                iu = 0;
            }
            issue();
        }
    };

    for (uint32_t par = 0; s_item[par] < items; par ^= 1) {
        const uint32_t item = s_item[par];
        const FwItem& g = s_desc[par];
        if (tid == boss) fetched = s_item[par ^ 1] < items ? gridDim.x + atomicAdd(w.counters, 1u) : items;
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
            if (issued - computed >= (uint32_t)NST - 1) asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
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
                    // 2^(127 - e) brings it to [1, 2); rows of zeros and tiny values, or of infinities, as they are
                    const uint32_t e = top >> 7;
                    const float f = e > 20 && e < 250 ? __uint_as_float((254u - e) << 23) : 1.0f;
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
            if (issued - computed >= (uint32_t)NST - 1) asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            fill(par);
            const int32_t kb = (int32_t)((k0 + u) * 64 + warp * 16);
            if (kb >= hi || kb + 16 <= lo) continue;
            const uint32_t st = ring + (computed % NST) * G::STAGE;
            // ---- S^T = K Q^T ----
            float s[NR][4], s2[NR][4];
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = s2[i][j] = 0.0f;
            {
                const uint32_t r = lane & 15, c0 = lane >> 4;
                if constexpr (Q8) {
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        uint32_t x[4];
                        fw_ldm(st + fw_at<RB>(r, k + c0), x);
                        const uint2 y0 = at_codes<M>(x[0], C{}), y1 = at_codes<M>(x[1], C{});
                        const uint2 y2 = at_codes<M>(x[2], C{}), y3 = at_codes<M>(x[3], C{});
                        const uint32_t a0[4] = {y0.x, y1.x, y0.y, y1.y}, a1[4] = {y2.x, y3.x, y2.y, y3.y};
#pragma unroll
                        for (int i = 0; i < NR; ++i) {
                            fw_mma<M>(s[i], a0, qf[k][i][0], qf[k][i][1]);
                            fw_mma<M>(s2[i], a1, qf[k + 1][i][0], qf[k + 1][i][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        uint32_t x[4];
                        fw_ldm(st + fw_at<RB>(r, 2 * k + c0), x);
#pragma unroll
                        for (int i = 0; i < NR; ++i) fw_mma<M>(k & 1 ? s2[i] : s[i], x, qf[k][i][0], qf[k][i][1]);
                    }
                }
            }
            // ---- weights: keys kb + lg (values 0, 1) and kb + lg + 8 (2, 3), rows 2 lq (0, 2) and 2 lq + 1 ----
            float rv[2] = {1.0f, 1.0f};
            if constexpr (Q8) {
                float ks[2], lv[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ks[j] = __uint_as_float(at_lds(st + 32 * RB + (lg + 8 * j) * 4));
                    const float vs = __uint_as_float(at_lds(st + 32 * RB + 64 + (lg + 8 * j) * 4));
                    lv[j] = log2f(vs);
                    rv[j] = 1.0f / vs;
                    if (kb + (int32_t)lg + 8 * j >= hi || kb + (int32_t)lg + 8 * j < lo || vs == 0.0f) {
                        // no key, or one whose page is missing: its codes are zeros
                        lv[j] = 0.0f;
                        rv[j] = 1.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i][j] = fmaf((s[i][j] + s2[i][j]) * rs[i][j & 1], ks[j >> 1], lv[j >> 1]);
            } else {
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i][j] = (s[i][j] + s2[i][j]) * a.scale_log2;
            }
            bool partial = false;  // some row does not see some key
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) partial |= kb < klo[i][j] || khi[i][j] - kb < 16;
            partial = __any_sync(0xffffffffu, partial);
            bool up = false;
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (partial) {
                        const int32_t key = kb + (int32_t)lg + 8 * (j >> 1);
                        if (key < klo[i][j & 1] || key >= khi[i][j & 1]) s[i][j] = -INFINITY;
                    }
                    up |= s[i][j] > m[i][j & 1] + 8.0f;
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float x = fmaxf(s[i][j], s[i][j + 2]);
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
            uint32_t pb[NR][2];
#pragma unroll
            for (int i = 0; i < NR; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = at_ex2(s[i][j] - ref[i][j & 1]);
                    l[i][j & 1] = fmaf(s[i][j], rv[j >> 1], l[i][j & 1]);
                }
                pb[i][0] = fw_movm(at_pack<M>(s[i][0], s[i][1]));
                pb[i][1] = fw_movm(at_pack<M>(s[i][2], s[i][3]));
            }
            // ---- O^T += V^T P^T ----
            const uint32_t sv = st + 16 * RB;
            if constexpr (Q8) {
                const uint32_t r = lane & 15, c0 = lane >> 4;
#pragma unroll
                for (int d = 0; d < KS; d += 2) {
                    uint32_t x[4];
                    fw_ldmt(sv + fw_at<RB>(r, d + c0), x);
                    // a dim's two keys side by side
                    const uint2 y0 = fw_codes_t(x[0], C{}), y1 = fw_codes_t(x[1], C{});
                    const uint2 y2 = fw_codes_t(x[2], C{}), y3 = fw_codes_t(x[3], C{});
                    const uint32_t a0[4] = {y0.x, y0.y, y1.x, y1.y}, a1[4] = {y2.x, y2.y, y3.x, y3.y};
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        fw_mma<M>(o[d][i], a0, pb[i][0], pb[i][1]);
                        fw_mma<M>(o[d + 1][i], a1, pb[i][0], pb[i][1]);
                    }
                }
            } else {
                const uint32_t r = (lane & 7) + (lane >> 4) * 8, c0 = (lane >> 3) & 1;
                constexpr uint32_t mask = std::is_same_v<T, bf16> ? 0x7F80u : 0x7C00u;
                bool odd = false;
#pragma unroll
                for (int d = 0; d < KS; ++d) {
                    uint32_t x[4];
                    fw_ldmt(sv + fw_at<RB>(r, 2 * d + c0), x);
                    if (partial) {  // infinities and NaN only to the rows that see them
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if ((x[j] & mask) == mask) { x[j] &= 0xFFFF0000u; odd = true; }
                            if ((x[j] & (mask << 16)) == (mask << 16)) { x[j] &= 0xFFFFu; odd = true; }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < NR; ++i) fw_mma<M>(o[d][i], x, pb[i][0], pb[i][1]);
                }
                if (partial && __any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int d = 0; d < KS; ++d)
                        for (uint32_t j = 0; j < 16; ++j)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                T v;
                                asm volatile("ld.shared.u16 %0, [%1];"
                                             : "=h"(reinterpret_cast<uint16_t&>(v))
                                             : "r"(sv + fw_at<RB>(j, 2 * d + half) + lg * 2)
                                             : "memory");
                                const float x = to_f32(v);
                                if (fabsf(x) <= 3.4028235e38f) continue;
#pragma unroll
                                for (int i = 0; i < NR; ++i)
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        if (kb + (int32_t)j >= klo[i][q] && kb + (int32_t)j < khi[i][q]) o[d][i][2 * half + q] += x;
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
        const bool whole = g.nch == 1;
        unsigned char* const part = w.slots + (size_t)item * w.slot_bytes;
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
                __stcg(reinterpret_cast<float4*>(part) + id, x);
                if (c == 0) __stcg(reinterpret_cast<float2*>(part + (size_t)ROWS * D * 4) + r, make_float2(ll != 0.0f ? top : 0.0f, ll));
            }
        }
        if (!whole) {
            const uint32_t item0 = item - g.ch;
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = atomicAdd(w.tickets + item0, 1u) == g.nch - 1;
                if (s_last) w.tickets[item0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                // 64 parts at a time: their m and l in shared memory, then the sums
                const unsigned char* const parts = w.slots + (size_t)item0 * w.slot_bytes;
                float2* const ml = reinterpret_cast<float2*>(sm + G::sum_off);  // [64][ROWS]
                constexpr uint32_t PER = (ROWS * (D / 4) + 127) / 128;  // of a thread
                float4 x[PER];
                float mm[PER], ll[PER];
#pragma unroll
                for (uint32_t k = 0; k < PER; ++k) {
                    x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    mm[k] = -INFINITY;
                    ll[k] = 0.0f;
                }
                for (uint32_t i0 = 0; i0 < g.nch; i0 += 64) {
                    const uint32_t m = min(g.nch - i0, 64u);
                    __syncthreads();
                    for (uint32_t i = tid; i < m * ROWS; i += 128) {
                        const uint32_t r = i % ROWS;
                        ml[i] = r < nrows ? __ldcg(reinterpret_cast<const float2*>(parts + (size_t)(i0 + i / ROWS) * w.slot_bytes +
                                                                                   (size_t)ROWS * D * 4) + r)
                                          : make_float2(0.0f, 0.0f);
                    }
                    __syncthreads();
#pragma unroll
                    for (uint32_t k = 0; k < PER; ++k) {
                        const uint32_t id = tid + k * 128, r = id / (D / 4);
                        if (r >= nrows) continue;
                        float top = mm[k];
                        for (uint32_t i = 0; i < m; ++i) {
                            const float2 v = ml[i * ROWS + r];
                            if (v.y != 0.0f) top = fmaxf(top, v.x);
                        }
                        const float f0 = mm[k] == -INFINITY ? 0.0f : at_ex2(mm[k] - top);
                        mm[k] = top;
                        ll[k] *= f0;
                        x[k].x *= f0;
                        x[k].y *= f0;
                        x[k].z *= f0;
                        x[k].w *= f0;
                        const unsigned char* p = parts + (size_t)i0 * w.slot_bytes + (size_t)id * 16;
#pragma unroll 8
                        for (uint32_t i = 0; i < m; ++i, p += w.slot_bytes) {
                            const float4 y = __ldcg(reinterpret_cast<const float4*>(p));
                            const float2 v = ml[i * ROWS + r];
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
        if (tid == boss) {
            s_item[par] = fetched;
            if (fetched < items) s_desc[par] = describe(fetched);
        }
        __syncthreads();
    }
    at_clear<T, D>(a, 128);
    // the last CTA leaves the counters as it found them
    if (tid == 0 && atomicAdd(w.counters + 1, 1u) == gridDim.x - 1) {
        w.counters[0] = 0;
        w.counters[1] = 0;
    }
}

}  // namespace xp
