// Rotary positions and the quantising paged cache: device code.
//
// Rotation. Pair (a, b) of a head turns by the angle of its position:
//   a' = m (a cos - b sin),  b' = m (a sin + b cos),  inverse: sin -> -sin.
// The angle is position * turns / 2^64 of a circle, an exact 64-bit product
// whose whole turns fall out of the top; what is left is rounded once, to 24
// bits of a turn, so position 10^6 is as exact as position 1. A thread makes
// the cosines and sines of its pairs once and applies them to all its heads.
//
// Cache rows. One warp per (token, kv head) holds the k row and the v row in
// registers, two vectors of W = dim / 64 values a lane, so the row's maximum
// is one warp reduction and the codes leave in the same pass.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace xp {

using bf16 = __nv_bfloat16;
struct int8c { int8_t v; };    // cache code types
struct fp8c { uint8_t v; };    // e4m3

template <class T> XP_DEV float to_f32(T x) { return (float)x; }
template <class T> XP_DEV T from_f32(float x);
template <> XP_DEV float from_f32<float>(float x) { return x; }
template <> XP_DEV __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> XP_DEV bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive values as one access (N * sizeof(T) of 1 to 16 bytes, aligned
// to its size)
template <class T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };
template <int N, class T> XP_DEV void load_f32(const T* p, float* x) {
    const Pack<T, N> r = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(r.v[i]);
}
template <int N, class T> XP_DEV void store_f32(T* p, const float* x) {
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = r;
}

struct RowsArg {
    void* data;
    int64_t ts, hs;  // token and head strides, elements
};
struct RopeArg {
    const unsigned long long* turns;
    const int32_t* positions;
    uint32_t rot;
    uint32_t interleaved;
    float magnitude;
    float sign;  // -1: inverse
};

// cos and sin of pair i at position `pos`, times the magnitude
XP_DEV void rope_angle(const RopeArg& r, int32_t pos, uint32_t i, float& c, float& s) {
    const long long part = (long long)((unsigned long long)(long long)pos * __ldg(r.turns + i));
    const float half_turns = (float)(int32_t)(part >> 32) * 0x1p-31f;
    sincospif(half_turns, &s, &c);
    c *= r.magnitude;
    s *= r.magnitude * r.sign;
}

// ---- rotary rows ----------------------------------------------------------
// A unit is VP pairs: two vectors of VP values of the head (half layout) or 2
// VP consecutive ones (interleaved); units past the rotated part copy 2 VP
// values. Thread = (token, unit) of `hpt` consecutive heads.
// VP > 1 needs rot / 2 and dim to be multiples of VP and 2 VP, and every row
// to be aligned to VP values; VP = 1 takes any strides and alignment.
template <class T, int VP>
__global__ void __launch_bounds__(256) rope_rows_kernel(RowsArg out, RowsArg in, RopeArg r, uint32_t tokens,
                                                        uint32_t heads, uint32_t dim, uint32_t hpt, uint32_t nunits,
                                                        bool copy_tail) {
    const uint32_t chunks = (heads + hpt - 1) / hpt;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t unit = (uint32_t)(id % nunits);
    const uint64_t rest = id / nunits;
    const uint32_t h0 = (uint32_t)(rest % chunks) * hpt;
    const uint64_t t = rest / chunks;
    if (t >= tokens) return;
    const uint32_t n = r.rot / 2, rot_units = n / VP;
    const T* src = static_cast<const T*>(in.data) + (int64_t)t * in.ts + (int64_t)h0 * in.hs;
    T* dst = static_cast<T*>(out.data) + (int64_t)t * out.ts + (int64_t)h0 * out.hs;
    const uint32_t nh = min(hpt, heads - h0);
    if (unit < rot_units) {
        const int32_t pos = __ldg(r.positions + t);
        float c[VP], s[VP];
#pragma unroll
        for (int i = 0; i < VP; ++i) rope_angle(r, pos, unit * VP + i, c[i], s[i]);
        const uint32_t a0 = r.interleaved ? 2 * unit * VP : unit * VP;
        const uint32_t b0 = r.interleaved ? a0 + VP : n + unit * VP;
#pragma unroll 4
        for (uint32_t h = 0; h < nh; ++h, src += in.hs, dst += out.hs) {
            float x[2 * VP], y[2 * VP];
            load_f32<VP>(src + a0, x);
            load_f32<VP>(src + b0, x + VP);
            if (r.interleaved) {
#pragma unroll
                for (int i = 0; i < VP; ++i) {
                    y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
                    y[2 * i + 1] = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < VP; ++i) {
                    y[i] = x[i] * c[i] - x[VP + i] * s[i];
                    y[VP + i] = x[i] * s[i] + x[VP + i] * c[i];
                }
            }
            store_f32<VP>(dst + a0, y);
            store_f32<VP>(dst + b0, y + VP);
        }
    } else if (copy_tail) {
        const uint32_t d = r.rot + (unit - rot_units) * 2 * VP;
        const bool second = d + VP < dim;
#pragma unroll 4
        for (uint32_t h = 0; h < nh; ++h, src += in.hs, dst += out.hs) {
            const Pack<T, VP> a = *reinterpret_cast<const Pack<T, VP>*>(src + d);
            Pack<T, VP> b{};
            if (second) b = *reinterpret_cast<const Pack<T, VP>*>(src + d + VP);
            *reinterpret_cast<Pack<T, VP>*>(dst + d) = a;
            if (second) *reinterpret_cast<Pack<T, VP>*>(dst + d + VP) = b;
        }
    }
}

// ---- cache rows -----------------------------------------------------------
struct PagesArg {
    void *k, *v;
    float *ks, *vs;
    uint64_t slots;        // num_pages * page_size
    uint32_t page_shift;   // log2 page_size
    uint32_t kv_heads;
};
// Row index (of head_dim values, and of scales) of a slot's head.
XP_DEV uint64_t page_row(const PagesArg& p, uint64_t slot, uint32_t head) {
    const uint64_t page = slot >> p.page_shift;
    return ((page * p.kv_heads + head) << p.page_shift) + (slot & ((1u << p.page_shift) - 1));
}

constexpr float CACHE_FLOOR = 0x1p-100f;  // smallest row maximum told from zero

// A row's 2 W values a lane (at lane_d[0] and lane_d[1]) into its place.
template <class C, int W>
XP_DEV void cache_row_store(C* row, float* scale, const float* x, const uint32_t* d) {
    if constexpr (sizeof(C) > 1) {
        store_f32<W>(row + d[0], x);
        store_f32<W>(row + d[1], x + W);
    } else {
        constexpr float Q = std::is_same_v<C, int8c> ? 127.0f : 448.0f;
        // the maximum as an integer: for |x| the order of the bits is the
        // order of the values, and an infinity or NaN is above them all
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        top = __reduce_max_sync(0xffffffffu, top);
        const bool finite = top < 0x7F800000u;
        const float m = fmaxf(__uint_as_float(top), CACHE_FLOOR);
        const float inv = finite ? __fdiv_rn(Q, m) : 0.0f;
        if ((threadIdx.x & 31) == 0) *scale = finite ? __fdiv_rn(m, Q) : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            Pack<uint8_t, W> r;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float y = finite ? x[j * W + i] * inv : 0.0f;
                if constexpr (std::is_same_v<C, int8c>) {
                    r.v[i] = (uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f));
                } else {
                    uint16_t two;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(y));
                    r.v[i] = (uint8_t)two;
                }
            }
            *reinterpret_cast<Pack<uint8_t, W>*>(reinterpret_cast<uint8_t*>(row) + d[j]) = r;
        }
    }
}

// One warp per (token, kv head). W = dim / 64 values in each of a lane's two
// vectors; with a rotation a lane's vectors are the two ends of its pairs.
template <class T, class C, int W>
__global__ void __launch_bounds__(256) kv_write_kernel(PagesArg p, RowsArg k, RowsArg v, const int64_t* slots,
                                                       uint32_t tokens, RopeArg r, bool rotate) {
    constexpr uint32_t DIM = 64 * W;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t id = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint64_t t = id / p.kv_heads;
    const uint32_t h = (uint32_t)(id % p.kv_heads);
    if (t >= tokens) return;
    const int64_t slot = __ldg(slots + t);
    if (slot < 0 || (uint64_t)slot >= p.slots) return;
    const T* kp = static_cast<const T*>(k.data) + (int64_t)t * k.ts + (int64_t)h * k.hs;
    const T* vp = static_cast<const T*>(v.data) + (int64_t)t * v.ts + (int64_t)h * v.hs;
    // the lane's vectors: contiguous pairs of vectors, except that a half-
    // layout rotation pairs vector j of the first half with j of the second
    uint32_t d[2] = {lane * 2 * W, lane * 2 * W + W};
    const uint32_t n = r.rot / 2;
    const bool turns = rotate && lane * W < n;
    if (turns && !r.interleaved) {
        d[0] = lane * W;
        d[1] = n + lane * W;
    }
    float kx[2 * W], vx[2 * W];
    load_f32<W>(kp + d[0], kx);
    load_f32<W>(kp + d[1], kx + W);
    load_f32<W>(vp + d[0], vx);
    load_f32<W>(vp + d[1], vx + W);
    if (turns) {
        const int32_t pos = __ldg(r.positions + t);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float c, s;
            rope_angle(r, pos, lane * W + i, c, s);
            float& a = r.interleaved ? kx[2 * i] : kx[i];
            float& b = r.interleaved ? kx[2 * i + 1] : kx[W + i];
            const float a1 = a * c - b * s, b1 = a * s + b * c;
            a = a1;
            b = b1;
        }
    }
    const uint64_t row = page_row(p, (uint64_t)slot, h);
    cache_row_store<C, W>(static_cast<C*>(p.k) + row * DIM, p.ks + row, kx, d);
    cache_row_store<C, W>(static_cast<C*>(p.v) + row * DIM, p.vs + row, vx, d);
}

// 4 codes of a word as fp32
XP_DEV void codes4(uint32_t w, int8c, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
}
XP_DEV void codes4(uint32_t w, fp8c, float* x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)(w >> (16 * i))));
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h2));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}

// Thread = 16 values of a (row, head), of k and of v.
template <class T, class C, int W>
__global__ void __launch_bounds__(256) kv_read_kernel(PagesArg p, RowsArg k, RowsArg v, const int64_t* slots,
                                                      uint32_t rows) {
    constexpr uint32_t DIM = 64 * W, PER = DIM / 16;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t part = (uint32_t)(id % PER) * 16;
    const uint64_t th = id / PER;
    const uint64_t t = th / p.kv_heads;
    const uint32_t h = (uint32_t)(th % p.kv_heads);
    if (t >= rows) return;
    const int64_t slot = __ldg(slots + t);
    const bool has = slot >= 0 && (uint64_t)slot < p.slots;
    const uint64_t row = page_row(p, has ? (uint64_t)slot : 0, h);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const C* src = static_cast<const C*>(side ? p.v : p.k) + row * DIM + part;
        const RowsArg& o = side ? v : k;
        T* dst = static_cast<T*>(o.data) + (int64_t)t * o.ts + (int64_t)h * o.hs + part;
        float x[16];
        if (!has) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.0f;
        } else if constexpr (sizeof(C) > 1) {
            load_f32<8>(src, x);
            load_f32<8>(src + 8, x + 8);
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(src);
            const float s = (side ? p.vs : p.ks)[row];
            codes4(w.x, C{}, x);
            codes4(w.y, C{}, x + 4);
            codes4(w.z, C{}, x + 8);
            codes4(w.w, C{}, x + 12);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= s;
        }
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += V) store_f32<V>(dst + i, x + i);
    }
}

}  // namespace xp
