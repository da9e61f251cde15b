// Attention of serving: whole prompts (packed) and new tokens over pages.
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = 2^(t_ij - m_i),  l_i = sum_j p_ij,
//   t_ij = (q_i . k_j) scale log2 e over the keys j that row i sees.
#pragma once
#include "serving.cuh"

namespace xp {

constexpr uint32_t SERVE_ERR_LENGTH = 1u;  // a kv length past its table row
constexpr uint32_t SERVE_ERR_PAGE = 2u;    // a page outside the cache
constexpr uint32_t SERVE_ERR_WAIT = 4u;    // a wait ran out
constexpr uint32_t SERVE_ERR_NEW = 8u;     // more new tokens than q_most

struct ServeAttnArgs {
    RowsArg out, q, k, v;      // k, v: packed only
    PagesArg pages;            // paged only (pages.k != nullptr)
    const int32_t* table;
    uint32_t table_width;
    const int32_t* kv_lens;
    const int32_t* starts;
    uint32_t batch, tokens, heads, kv_heads, group, q_most, window;
    float scale_log2;          // scale * log2 e
    float* lse;
    uint32_t* err;
};

// Sequence b: its first q row, new tokens and keys. Whatever the device arrays
// hold, q0 + nq <= tokens and nkv <= the table row's rows.
struct Seq { uint32_t q0, nq, nkv; };
XP_DEV Seq seq_of(const ServeAttnArgs& a, uint32_t b) {
    Seq s;
    const int32_t lo = __ldg(a.starts + b), hi = __ldg(a.starts + b + 1);
    s.q0 = (uint32_t)min(max(lo, 0), (int32_t)a.tokens);
    s.nq = (uint32_t)max(min(max(hi, 0), (int32_t)a.tokens) - (int32_t)s.q0, 0);
    if (a.pages.k) {
        const uint64_t most = (uint64_t)a.table_width << a.pages.page_shift;
        const int32_t n = max(__ldg(a.kv_lens + b), 0);
        s.nkv = (uint32_t)min((uint64_t)n, most);
        if ((uint64_t)n > most) atomicOr(a.err, SERVE_ERR_LENGTH);
        if (s.nq > a.q_most) {
            s.nq = a.q_most;
            atomicOr(a.err, SERVE_ERR_NEW);
        }
    } else {
        s.nkv = s.nq;
    }
    return s;
}

// One CTA per (token, head), one warp per key.
template <class T, class C, int W>
__global__ void __launch_bounds__(128) attn_rows_kernel(const __grid_constant__ ServeAttnArgs a) {
    constexpr uint32_t DIM = 64 * W, PER = 2 * W;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t token = blockIdx.x, head = blockIdx.y, kvh = head / a.group;
    __shared__ float s_m[4], s_l[4], s_o[4][DIM];
    __shared__ uint32_t s_b;
    if (tid == 0) {
        uint32_t lo = 0, hi = a.batch;  // first b with starts[b + 1] > token
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (__ldg(a.starts + mid + 1) > (int32_t)token) hi = mid;
            else lo = mid + 1;
        }
        s_b = lo;
    }
    __syncthreads();
    const uint32_t b = s_b;
    const Seq s = b < a.batch ? seq_of(a, b) : Seq{0, 0, 0};
    float q[PER], o[PER], m = -INFINITY, l = 0.0f;
    load_f32<PER>(static_cast<const T*>(a.q.data) + token * a.q.ts + head * a.q.hs + lane * PER, q);
#pragma unroll
    for (int i = 0; i < (int)PER; ++i) o[i] = 0.0f;
    const int64_t pos = (int64_t)s.nkv - s.nq + (token - s.q0);
    if (token >= s.q0 && token - s.q0 < s.nq && pos >= 0) {
        const int64_t first = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0;
        for (int64_t j = first + warp; j <= pos; j += 4) {
            float k[PER], v[PER], ks = 1.0f, vs = 1.0f;
            if (a.pages.k) {
                const int32_t page = __ldg(a.table + (uint64_t)b * a.table_width + (j >> a.pages.page_shift));
                const uint64_t slot = ((uint64_t)(uint32_t)page << a.pages.page_shift) +
                                      (j & ((1u << a.pages.page_shift) - 1));
                if (page < 0 || slot >= a.pages.slots) {
                    if (lane == 0) atomicOr(a.err, SERVE_ERR_PAGE);
#pragma unroll
                    for (int i = 0; i < (int)PER; ++i) k[i] = v[i] = 0.0f;
                } else {
                    const uint64_t row = page_row(a.pages, slot, kvh);
                    const C* kp = static_cast<const C*>(a.pages.k) + row * DIM + lane * PER;
                    const C* vp = static_cast<const C*>(a.pages.v) + row * DIM + lane * PER;
                    if constexpr (sizeof(C) > 1) {
                        load_f32<PER>(kp, k);
                        load_f32<PER>(vp, v);
                    } else {
                        float x[4];
                        const Pack<uint8_t, PER> kc = *reinterpret_cast<const Pack<uint8_t, PER>*>(kp);
                        const Pack<uint8_t, PER> vc = *reinterpret_cast<const Pack<uint8_t, PER>*>(vp);
                        ks = a.pages.ks[row];
                        vs = a.pages.vs[row];
#pragma unroll
                        for (int i = 0; i < (int)PER; ++i) {
                            codes4(kc.v[i], C{}, x);
                            k[i] = x[0] * ks;
                            codes4(vc.v[i], C{}, x);
                            v[i] = x[0] * vs;
                        }
                    }
                }
            } else {
                load_f32<PER>(static_cast<const T*>(a.k.data) + (s.q0 + j) * a.k.ts + kvh * a.k.hs + lane * PER, k);
                load_f32<PER>(static_cast<const T*>(a.v.data) + (s.q0 + j) * a.v.ts + kvh * a.v.hs + lane * PER, v);
            }
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < (int)PER; ++i) t += q[i] * k[i];
            t = warp_sum(t) * a.scale_log2;
            const float mn = fmaxf(m, t);
            if (t == -INFINITY) continue;  // an infinite key that points away: no weight
            const float w = exp2f(m - mn), p = exp2f(t - mn);
            l = l * w + p;
#pragma unroll
            for (int i = 0; i < (int)PER; ++i) o[i] = o[i] * w + p * v[i];
            m = mn;
        }
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < (int)PER; ++i) s_o[warp][lane * PER + i] = o[i];
    __syncthreads();
    float mm = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3])), ll = 0.0f, w[4];
    const bool any = !(s_l[0] == 0.0f && s_l[1] == 0.0f && s_l[2] == 0.0f && s_l[3] == 0.0f);
    for (int i = 0; i < 4; ++i) {
        w[i] = s_l[i] == 0.0f ? 0.0f : exp2f(s_m[i] - mm);
        ll += w[i] * s_l[i];
    }
    T* op = static_cast<T*>(a.out.data) + token * a.out.ts + head * a.out.hs;
    for (uint32_t d = tid; d < DIM; d += 128) {
        float x = 0.0f;
        for (int i = 0; i < 4; ++i) x += w[i] * s_o[i][d];
        op[d] = from_f32<T>(any ? x / ll : 0.0f);
    }
    if (a.lse && tid == 0) a.lse[(uint64_t)token * a.heads + head] = any ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace xp
