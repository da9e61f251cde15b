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
// The four warps of a CTA take the keys of a unit of 64 in turn and add their
// sums in shared memory; CTAs have equal shares of all units, whatever the
// lengths, and of a sequence that several share the last to finish adds the
// parts, in their order.
#pragma once
#include "serving_tile.cuh"

namespace xp {

template <class T, class C, int W, int NR> struct FwCfg {
    static constexpr int D = 64 * W;
    static constexpr bool Q8 = sizeof(C) == 1;
    static constexpr int RB = D * (int)sizeof(C);            // bytes of a row
    static constexpr int STAGE = 2 * 16 * RB + (Q8 ? 128 : 0);  // 16 keys: K, V, scales
    static constexpr int NST = STAGE > 8500 ? 2 : STAGE > 4300 ? 3 : STAGE > 2200 ? 3 : 6;
    static constexpr int MERGE = 4 * 8 * NR * (D + 4) * 4;   // the warps' sums, and their m and l
    static constexpr int RING = 4 * NST * STAGE > MERGE ? 4 * NST * STAGE : MERGE;
    static constexpr int smem = RING > AT_MAX_BATCH * 4 ? RING : AT_MAX_BATCH * 4;
    static constexpr int CTAS = smem > 116000 ? 1 : smem > 76000 || W * NR > 4 ? 2 : W == 4 ? 3 : 4;  // of an SM
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
// where 16 bytes c of row r of a stage lie: eight rows' equal chunks in eight bank groups
template <int RB> XP_DEV uint32_t fw_at(uint32_t r, uint32_t c) {
    if constexpr (RB >= 128) return r * RB + ((c & ~7u) << 4) + (((c ^ r) & 7) << 4);
    else return (r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (r >> 1)) & 7) * 16;
}

template <class T, class C, int W, int NR>
__global__ void __launch_bounds__(128, (FwCfg<T, C, W, NR>::CTAS))
attn_few_kernel(const __grid_constant__ ServeAttnArgs a, const __grid_constant__ AtWork w, uint32_t* tickets) {
    using G = FwCfg<T, C, W, NR>;
    constexpr int D = G::D, RB = G::RB, NST = G::NST, KS = D / 16, ROWS = 8 * NR;
    constexpr bool Q8 = G::Q8;
    extern __shared__ __align__(1024) unsigned char sm[];
    __shared__ AtPlan s_plan;
    __shared__ uint32_t s_sums[32], s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lg = lane >> 2, lq = lane & 3;
    const uint32_t ring = smem_u32(sm) + warp * (NST * G::STAGE);
    at_clear<T, D>(a, 128);
    at_make_plan<128>(a, w, reinterpret_cast<uint32_t*>(sm), s_sums, &s_plan);
    __syncthreads();
    AtWalk walk;
    walk.start(s_plan);
    AtSeg g;
    while (walk.next(a, w, g)) {
        // this lane's rows: 8 i + lg as a row of Q, 8 i + 2 lq and the next as columns of S^T and O^T
        const int32_t first = (int32_t)g.s.nkv - (int32_t)g.s.nq;
        const uint32_t nrows = g.s.nq * a.group;
        uint32_t qf[KS][NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const uint32_t r = 8 * i + lg, tok = r / a.group, h = g.h * a.group + (r - tok * a.group);
            const T* qp = static_cast<const T*>(a.q.data) + (int64_t)(g.s.q0 + tok) * a.q.ts + (int64_t)h * a.q.hs;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                // the values that stand where the codes of a key's word stand (8-bit), or in order
                qf[s][i][0] = qf[s][i][1] = 0;
                if (r < nrows) {
                    qf[s][i][0] = __ldg(reinterpret_cast<const uint32_t*>(qp + s * 16 + (Q8 ? 4 * lq : 2 * lq)));
                    qf[s][i][1] = __ldg(reinterpret_cast<const uint32_t*>(qp + s * 16 + (Q8 ? 4 * lq + 2 : 2 * lq + 8)));
                }
            }
        }
        int32_t klo[NR][2], khi[NR][2];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = 8 * i + 2 * lq + j;
                const int32_t pos = first + (int32_t)(r / a.group);
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
        // ---- the ring ----
        const int32_t lo = g.lo, hi = g.hi;
        const int32_t* const table = a.table + (uint64_t)g.b * a.table_width;
        auto key_of = [&](uint32_t u) { return (int32_t)((g.k0 + u) * 64 + warp * 16); };
        auto page_of = [&](uint32_t u) -> int32_t {  // lane & 15: the key
            const int32_t key = key_of(u) + (int32_t)(lane & 15);
            return u < g.n && key >= lo && key < hi ? __ldg(table + (key >> a.pages.page_shift)) : -1;
        };
        int32_t page = page_of(0);
        auto issue = [&](uint32_t u) {
            const int32_t kb = key_of(u);
            if (u < g.n && kb < hi && kb + 16 > lo) {
                const int32_t key = kb + (int32_t)(lane & 15);
                uint32_t row = AT_NONE;
                if (key >= lo && key < hi) {
                    const uint64_t slot = ((uint64_t)(uint32_t)page << a.pages.page_shift) +
                                          ((uint32_t)key & ((1u << a.pages.page_shift) - 1));
                    if (page < 0 || slot >= a.pages.slots) atomicOr(a.err, SERVE_ERR_PAGE);
                    else row = (uint32_t)page_row(a.pages, slot, g.h);
                }
                const uint32_t st = ring + (u % NST) * G::STAGE;
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
            page = page_of(u + 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll 1
        for (uint32_t u = 0; u < (uint32_t)NST - 1; ++u) issue(u);
#pragma unroll 1
        for (uint32_t u = 0; u < g.n; ++u) {
            asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
            __syncwarp();
            issue(u + NST - 1);
            const int32_t kb = key_of(u);
            if (kb >= hi || kb + 16 <= lo) continue;
            const uint32_t st = ring + (u % NST) * G::STAGE;
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
                        const uint2 y0 = at_codes<T>(x[0], C{}), y1 = at_codes<T>(x[1], C{});
                        const uint2 y2 = at_codes<T>(x[2], C{}), y3 = at_codes<T>(x[3], C{});
                        const uint32_t a0[4] = {y0.x, y1.x, y0.y, y1.y}, a1[4] = {y2.x, y3.x, y2.y, y3.y};
#pragma unroll
                        for (int i = 0; i < NR; ++i) {
                            fw_mma<T>(s[i], a0, qf[k][i][0], qf[k][i][1]);
                            fw_mma<T>(s2[i], a1, qf[k + 1][i][0], qf[k + 1][i][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        uint32_t x[4];
                        fw_ldm(st + fw_at<RB>(r, 2 * k + c0), x);
#pragma unroll
                        for (int i = 0; i < NR; ++i) fw_mma<T>(k & 1 ? s2[i] : s[i], x, qf[k][i][0], qf[k][i][1]);
                    }
                }
            }
            // ---- weights: keys kb + lg (values 0, 1) and kb + lg + 8 (2, 3), rows 2 lq (0, 2) and 2 lq + 1 ----
            float rv[2] = {1.0f, 1.0f};
            if constexpr (Q8) {
                float ks[2], lv[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ks[j] = __uint_as_float(at_lds(st + 32 * RB + (lg + 8 * j) * 4)) * a.scale_log2;
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
                    for (int j = 0; j < 4; ++j) s[i][j] = fmaf(s[i][j] + s2[i][j], ks[j >> 1], lv[j >> 1]);
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
                pb[i][0] = fw_movm(at_pack<T>(s[i][0], s[i][1]));
                pb[i][1] = fw_movm(at_pack<T>(s[i][2], s[i][3]));
            }
            // ---- O^T += V^T P^T ----
            const uint32_t sv = st + 16 * RB;
            if constexpr (Q8) {
                const uint32_t r = lane & 15, c0 = lane >> 4;
#pragma unroll
                for (int d = 0; d < KS; d += 2) {
                    uint32_t x[4];
                    fw_ldmt(sv + fw_at<RB>(r, d + c0), x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = __byte_perm(x[j], 0, 0x3120);  // a dim's two keys side by side
                    const uint2 y0 = at_codes<T>(x[0], C{}), y1 = at_codes<T>(x[1], C{});
                    const uint2 y2 = at_codes<T>(x[2], C{}), y3 = at_codes<T>(x[3], C{});
                    const uint32_t a0[4] = {y0.x, y0.y, y1.x, y1.y}, a1[4] = {y2.x, y2.y, y3.x, y3.y};
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        fw_mma<T>(o[d][i], a0, pb[i][0], pb[i][1]);
                        fw_mma<T>(o[d + 1][i], a1, pb[i][0], pb[i][1]);
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
                    for (int i = 0; i < NR; ++i) fw_mma<T>(o[d][i], x, pb[i][0], pb[i][1]);
                }
                if (partial && __any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int d = 0; d < KS; ++d)
                        for (uint32_t j = 0; j < 16; ++j)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint32_t dim = lg + 8 * half;
                                T v;
                                asm volatile("ld.shared.u16 %0, [%1];"
                                             : "=h"(reinterpret_cast<uint16_t&>(v))
                                             : "r"(sv + fw_at<RB>(j, 2 * d + half) + lg * 2)
                                             : "memory");
                                (void)dim;
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
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // ---- the warps' sums, one after the other ----
        __syncthreads();
        float* const so = reinterpret_cast<float*>(sm);                 // [4][ROWS][D]
        float2* const sml = reinterpret_cast<float2*>(sm + 4 * ROWS * D * 4);  // [4][ROWS] m, l
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = l[i][j];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                const uint32_t r = 8 * i + 2 * lq + j;
                if (lg == 0) sml[warp * ROWS + r] = make_float2(ref[i][j], x);
                if (r < nrows) {
#pragma unroll
                    for (int d = 0; d < KS; ++d) {
                        float* p = so + (warp * ROWS + r) * D + d * 16;
                        p[Q8 ? 2 * lg : lg] = o[d][i][j];
                        p[Q8 ? 2 * lg + 1 : lg + 8] = o[d][i][j + 2];
                    }
                }
            }
        __syncthreads();
        const bool whole = g.kind == AT_FULL;
        const uint32_t slot = 2 * blockIdx.x + (g.kind == AT_FIRST ? 1 : 0);
        unsigned char* const part = w.slots + (size_t)slot * w.slot_bytes;
        auto emit = [&](uint32_t r, uint32_t c, float4 x, float mm, float ll) {
            const float inv = ll != 0.0f ? 1.0f / ll : 0.0f;
            const uint32_t tok = r / a.group, h = g.h * a.group + (r - tok * a.group);
            uint2 y;
            y.x = at_pack<T>(x.x * inv, x.y * inv);
            y.y = at_pack<T>(x.z * inv, x.w * inv);
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out.data) + (int64_t)(g.s.q0 + tok) * a.out.ts + (int64_t)h * a.out.hs +
                                      4 * c) = y;
            if (a.lse && c == 0)
                a.lse[(uint64_t)(g.s.q0 + tok) * a.heads + h] = ll != 0.0f ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
        };
        for (uint32_t id = tid; id < nrows * (D / 4); id += 128) {
            const uint32_t r = id / (D / 4), c = id % (D / 4);
            float2 v[4];
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = sml[i * ROWS + r];
                if (v[i].y != 0.0f) mm = fmaxf(mm, v[i].x);
            }
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (v[i].y == 0.0f) continue;
                const float f = at_ex2(v[i].x - mm);
                const float4 y = *reinterpret_cast<const float4*>(so + (i * ROWS + r) * D + 4 * c);
                ll += f * v[i].y;
                x.x += f * y.x;
                x.y += f * y.y;
                x.z += f * y.z;
                x.w += f * y.w;
            }
            if (whole) {
                emit(r, c, x, mm, ll);
            } else {
                __stcg(reinterpret_cast<float4*>(part) + id, x);
                if (c == 0) __stcg(reinterpret_cast<float2*>(part + (size_t)ROWS * D * 4) + r, make_float2(mm, ll));
            }
        }
        if (!whole) {
            // the CTAs that have this sequence: those of its first and last unit, and all between
            const uint64_t u0 = g.at + w.cost, u1 = u0 + g.all - 1, total = s_plan.total, n = s_plan.ctas;
            const uint32_t c0 = (uint32_t)(((u0 + 1) * n + total - 1) / total - 1);
            const uint32_t c1 = (uint32_t)(((u1 + 1) * n + total - 1) / total - 1);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = atomicAdd(tickets + c0, 1u) == c1 - c0;
                if (s_last) tickets[c0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                auto part_of = [&](uint32_t c) { return w.slots + (size_t)(c == c0 ? 2 * c + 1 : 2 * c) * w.slot_bytes; };
                for (uint32_t id = tid; id < nrows * (D / 4); id += 128) {
                    const uint32_t r = id / (D / 4), c = id % (D / 4);
                    float mm = -INFINITY, ll = 0.0f;
#pragma unroll 8
                    for (uint32_t i = c0; i <= c1; ++i) {
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(part_of(i) + (size_t)ROWS * D * 4) + r);
                        if (v.y != 0.0f) mm = fmaxf(mm, v.x);
                    }
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (uint32_t i = c0; i <= c1; ++i) {
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(part_of(i) + (size_t)ROWS * D * 4) + r);
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(part_of(i)) + id);
                        const float f = v.y != 0.0f ? at_ex2(v.x - mm) : 0.0f;
                        ll += f * v.y;
                        x.x += f * y.x;
                        x.y += f * y.y;
                        x.z += f * y.z;
                        x.w += f * y.w;
                    }
                    emit(r, c, x, mm, ll);
                }
            }
        }
        __syncthreads();
    }
}

}  // namespace xp
