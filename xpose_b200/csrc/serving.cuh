// Rotary positions and the quantising paged cache: device code.
//
// Rotation. Pair (a, b) of a head turns by the angle of its position:
//   a' = m (a cos - b sin),  b' = m (a sin + b cos),  inverse: sin -> -sin.
// The angle is position * turns / 2^64 of a circle, an exact 64-bit product
// whose whole turns fall out of the top; what is left is rounded once, to 24
// bits of a turn, so position 10^6 is as exact as position 1. A thread makes
// the cosines and sines of its pairs once and applies them to all its heads.
//
// Cache rows. dim / 8 lanes hold a row of k and one of v in registers, two
// vectors of four values a lane, so a row's maximum is a few shuffles and the
// codes leave in the same pass.
//
// All three are bound by memory: 16381 tokens x 32 heads of 128 rotated in 51 us
// (5.3 TB/s), 8191 x 8 rows of 128 written in e4m3 and 32768 x 8 read in 52 us (4.9
// TB/s for the two launches); 64 rows take 2.5 us on the device, 3.3 a call.
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

// 32 bytes of values as one access (`side`: they lie side by side, aligned to
// 32) or as two vectors
struct Raw32 { uint32_t w[8]; };
XP_DEV Raw32 load_raw32(const void* a, const void* b, bool side) {
    Raw32 r;
    if (side) {
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"  // in order with pdl_wait()
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                       "=r"(r.w[7])
                     : "l"(a)
                     : "memory");
    } else {
        const uint4 x = *static_cast<const uint4*>(a), y = *static_cast<const uint4*>(b);
        r = Raw32{{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}};
    }
    return r;
}
XP_DEV void store_raw32(void* a, void* b, const Raw32& r, bool side) {
    if (side) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(a), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                     "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                     : "memory");
    } else {
        *static_cast<uint4*>(a) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
        *static_cast<uint4*>(b) = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
    }
}
// its 32 / sizeof(T) values
template <class T> XP_DEV float raw_get(const Raw32& r, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
    else if constexpr (std::is_same_v<T, bf16>) return i & 1 ? bf16_hi(r.w[i / 2]) : bf16_lo(r.w[i / 2]);
    else return __half2float(__ushort_as_half((unsigned short)(r.w[i / 2] >> (16 * (i & 1)))));
}
template <class T> XP_DEV void raw_put2(Raw32& r, int i, float x, float y) {  // values i and i + 1, i even
    if constexpr (sizeof(T) == 4) {
        r.w[i] = __float_as_uint(x);
        r.w[i + 1] = __float_as_uint(y);
    } else if constexpr (std::is_same_v<T, bf16>) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.w[i / 2]) : "f"(y), "f"(x));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r.w[i / 2]) : "f"(y), "f"(x));
    }
}

// Words that other kernels write, positions and lengths and the like. Not by
// the read-only path: a grid that starts under the kernel before it is not
// alone with them, even if it reads them only once that one has ended. In order
// with pdl_wait(), as volatile.
XP_DEV int32_t ld_now(const int32_t* p) {
    int32_t x;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(x) : "l"(p));
    return x;
}
template <class T> XP_DEV T ld_now(const T* p) {
    static_assert(sizeof(T) == 8);
    T x;
    asm volatile("ld.global.b64 %0, [%1];" : "=l"(x) : "l"(p));
    return x;
}

// ... and data that is read once, past the L1 cache
XP_DEV uint4 ld_once(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
XP_DEV float4 ld_once(const float4* p) {
    const uint4 v = ld_once(reinterpret_cast<const uint4*>(p));
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
XP_DEV float2 ld_once(const float2* p) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}
XP_DEV uint32_t ld_once(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
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
    const long long part = (long long)((unsigned long long)(long long)pos * ld_now(r.turns + i));
    const float half_turns = (float)(int32_t)(part >> 32) * 0x1p-31f;
    sincospif(half_turns, &s, &c);
    c *= r.magnitude;
    s *= r.magnitude * r.sign;
}

// ---- rotary rows ----------------------------------------------------------
// A unit is VP pairs: two vectors of VP values of the head (half layout) or 2
// VP consecutive ones (interleaved); units past the rotated part copy 2 VP
// values. Thread = (token, unit) of `hpt` consecutive heads.
// VP > 1 needs rot / 2 and dim to be multiples of VP, and every row to be
// aligned to VP values; VP = 1 takes any strides and alignment. `side`: rows
// are aligned to 2 VP values, so that values side by side move in one access
// of 32 bytes (a whole sector; two of 16 took 75 us where this takes 51, 16381
// tokens x 32 heads of 128 in bf16). Three CTAs an SM: two took 60 us, four 69.
template <class T, int VP>
__global__ void __launch_bounds__(256, 3) rope_rows_kernel(RowsArg out, RowsArg in, RopeArg r, uint32_t tokens,
                                                        uint32_t heads, uint32_t dim, uint32_t hpt, uint32_t nunits,
                                                        bool copy_tail, bool side) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t chunks = (heads + hpt - 1) / hpt;
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, rest = id / nunits, unit = id - rest * nunits;
    const uint32_t t = rest / chunks, h0 = (rest - t * chunks) * hpt;
    if (t >= tokens) return;
    const uint32_t n = r.rot / 2, rot_units = n / VP;
    const T* src = static_cast<const T*>(in.data) + (int64_t)t * in.ts + (int64_t)h0 * in.hs;
    T* dst = static_cast<T*>(out.data) + (int64_t)t * out.ts + (int64_t)h0 * out.hs;
    const uint32_t nh = min(hpt, heads - h0);
    if (unit < rot_units) {
        const int32_t pos = ld_now(r.positions + t);
        float c[VP], s[VP];
#pragma unroll
        for (int i = 0; i < VP; ++i) rope_angle(r, pos, unit * VP + i, c[i], s[i]);
        const uint32_t a0 = r.interleaved ? 2 * unit * VP : unit * VP;
        const uint32_t b0 = r.interleaved ? a0 + VP : n + unit * VP;
        if constexpr (VP > 1) {
            const bool both = side && r.interleaved;
            constexpr uint32_t B = 4;  // heads whose loads are under way together
            for (uint32_t h = 0; h < nh; h += B) {
                Raw32 x[B];
#pragma unroll
                for (uint32_t j = 0; j < B; ++j)
                    if (h + j < nh) x[j] = load_raw32(src + (h + j) * in.hs + a0, src + (h + j) * in.hs + b0, both);
#pragma unroll
                for (uint32_t j = 0; j < B; ++j) {
                    if (h + j >= nh) break;
                    Raw32 y;
                    if (r.interleaved) {
#pragma unroll
                        for (int i = 0; i < VP; ++i) {
                            const float p = raw_get<T>(x[j], 2 * i), q = raw_get<T>(x[j], 2 * i + 1);
                            raw_put2<T>(y, 2 * i, p * c[i] - q * s[i], p * s[i] + q * c[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < VP; i += 2) {
                            const float p0 = raw_get<T>(x[j], i), q0 = raw_get<T>(x[j], VP + i);
                            const float p1 = raw_get<T>(x[j], i + 1), q1 = raw_get<T>(x[j], VP + i + 1);
                            raw_put2<T>(y, i, p0 * c[i] - q0 * s[i], p1 * c[i + 1] - q1 * s[i + 1]);
                            raw_put2<T>(y, VP + i, p0 * s[i] + q0 * c[i], p1 * s[i + 1] + q1 * c[i + 1]);
                        }
                    }
                    store_raw32(dst + (h + j) * out.hs + a0, dst + (h + j) * out.hs + b0, y, both);
                }
            }
        } else {
            for (uint32_t h = 0; h < nh; ++h, src += in.hs, dst += out.hs) {
                const float p = to_f32(src[a0]), q = to_f32(src[b0]);
                dst[a0] = from_f32<T>(p * c[0] - q * s[0]);
                dst[b0] = from_f32<T>(p * s[0] + q * c[0]);
            }
        }
    } else if (copy_tail) {
        const uint32_t d = r.rot + (unit - rot_units) * 2 * VP;
        const bool second = d + VP < dim;
        if constexpr (VP > 1) {
            constexpr uint32_t B = 4;
            for (uint32_t h = 0; h < nh; h += B) {
                Raw32 x[B];
#pragma unroll
                for (uint32_t j = 0; j < B; ++j)
                    if (h + j < nh) {
                        const T* p = src + (h + j) * in.hs + d;
                        x[j] = load_raw32(p, second ? p + VP : p, side && second);
                    }
#pragma unroll
                for (uint32_t j = 0; j < B; ++j) {
                    if (h + j >= nh) break;
                    T* p = dst + (h + j) * out.hs + d;
                    if (second) store_raw32(p, p + VP, x[j], side);
                    else *reinterpret_cast<uint4*>(p) = make_uint4(x[j].w[0], x[j].w[1], x[j].w[2], x[j].w[3]);
                }
            }
        } else {
            for (uint32_t h = 0; h < nh; ++h, src += in.hs, dst += out.hs) {
                dst[d] = src[d];
                if (second) dst[d + 1] = src[d + 1];
            }
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
// Values with a scale below this count as zeros in attention: those of a row
// whose maximum is at most CACHE_FLOOR, and of scales that have no normal inverse.
constexpr float CACHE_NOTHING = 0x1p-106f;
static_assert(CACHE_FLOOR / 127.0f < CACHE_NOTHING, "int8 has the larger scales");

// A lane's 8 values of a row, four at d[0] and four at d[1], into its place;
// LANES lanes hold the row.
template <class C, int LANES>
XP_DEV void cache_row_store(C* row, float* scale, const float* x, const uint32_t* d, bool live) {
    if constexpr (sizeof(C) > 1) {
        if (!live) return;
        if (d[1] == d[0] + 4) {
            store_f32<8>(row + d[0], x);
        } else {
            store_f32<4>(row + d[0], x);
            store_f32<4>(row + d[1], x + 4);
        }
    } else {
        constexpr float Q = std::is_same_v<C, int8c> ? 127.0f : 448.0f;
        // the maximum as an integer: for |x| the order of the bits is the
        // order of the values, and an infinity or NaN is above them all
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (!live) return;
        const bool finite = top < 0x7F800000u;
        const float m = fmaxf(__uint_as_float(top), CACHE_FLOOR);
        const float inv = finite ? __fdiv_rn(Q, m) : 0.0f;
        if (threadIdx.x % LANES == 0) *scale = finite ? __fdiv_rn(m, Q) : __uint_as_float(0x7FC00000u);
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y = finite ? x[j * 4 + i] * inv : 0.0f;
                if constexpr (std::is_same_v<C, int8c>) {
                    b[i] = (uint32_t)__float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f)) & 0xFFu;
                } else {
                    uint16_t two;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(y));
                    b[i] = two & 0xFFu;
                }
            }
            w[j] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        }
        uint8_t* const p = reinterpret_cast<uint8_t*>(row);
        if (d[1] == d[0] + 4) {
            *reinterpret_cast<uint2*>(p + d[0]) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(p + d[0]) = w[0];
            *reinterpret_cast<uint32_t*>(p + d[1]) = w[1];
        }
    }
}

// dim / 8 lanes per (token, kv head). A lane's two vectors of four lie side by
// side, except that a half-layout rotation pairs four of the first half with
// the four that turn with them.
template <class T, class C, int W>
__global__ void __launch_bounds__(256) kv_write_kernel(PagesArg p, RowsArg k, RowsArg v, const int64_t* slots,
                                                       uint32_t tokens, RopeArg r, bool rotate) {
    constexpr uint32_t DIM = 64 * W, LANES = DIM / 8;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t part = threadIdx.x % LANES, id = (blockIdx.x * 256 + threadIdx.x) / LANES;
    const uint32_t t = id / p.kv_heads, h = id - t * p.kv_heads;
    const int64_t slot = t < tokens ? ld_now(slots + t) : -1;
    const bool live = slot >= 0 && (uint64_t)slot < p.slots;  // others only take part in the shuffles
    uint32_t d[2] = {part * 8, part * 8 + 4};
    const uint32_t n = r.rot / 2;
    const bool turns = rotate && part * 4 < n;
    if (turns && !r.interleaved) {
        d[0] = part * 4;
        d[1] = n + part * 4;
    }
    float kx[8] = {}, vx[8] = {};
    if (live) {
        const T* kp = static_cast<const T*>(k.data) + (int64_t)t * k.ts + (int64_t)h * k.hs;
        const T* vp = static_cast<const T*>(v.data) + (int64_t)t * v.ts + (int64_t)h * v.hs;
        if (sizeof(T) == 2 && d[1] == d[0] + 4) {
            load_f32<8>(kp + d[0], kx);
            load_f32<8>(vp + d[0], vx);
        } else {
            load_f32<4>(kp + d[0], kx);
            load_f32<4>(kp + d[1], kx + 4);
            load_f32<4>(vp + d[0], vx);
            load_f32<4>(vp + d[1], vx + 4);
        }
        if (turns) {
            const int32_t pos = ld_now(r.positions + t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float c, s;
                rope_angle(r, pos, part * 4 + i, c, s);
                const float a = r.interleaved ? kx[2 * i] : kx[i], b = r.interleaved ? kx[2 * i + 1] : kx[4 + i];
                const float a1 = a * c - b * s, b1 = a * s + b * c;
                if (r.interleaved) {
                    kx[2 * i] = a1;
                    kx[2 * i + 1] = b1;
                } else {
                    kx[i] = a1;
                    kx[4 + i] = b1;
                }
            }
        }
    }
    const uint64_t row = live ? page_row(p, (uint64_t)slot, h) : 0;
    cache_row_store<C, LANES>(static_cast<C*>(p.k) + row * DIM, p.ks + row, kx, d, live);
    cache_row_store<C, LANES>(static_cast<C*>(p.v) + row * DIM, p.vs + row, vx, d, live);
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
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, part = id % PER * 16, th = id / PER;
    const uint32_t t = th / p.kv_heads, h = th - t * p.kv_heads;
    if (t >= rows) return;
    const int64_t slot = ld_now(slots + t);
    const bool has = slot >= 0 && (uint64_t)slot < p.slots;
    const uint64_t row = page_row(p, has ? (uint64_t)slot : 0, h);
    // both sides' codes and scales under way together
    Pack<C, 16> c[2];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const C* src = static_cast<const C*>(side ? p.v : p.k) + row * DIM + part;
        if (has) {
            if constexpr (sizeof(C) > 1) {
                reinterpret_cast<uint4*>(&c[side])[0] = reinterpret_cast<const uint4*>(src)[0];
                reinterpret_cast<uint4*>(&c[side])[1] = reinterpret_cast<const uint4*>(src)[1];
            } else {
                *reinterpret_cast<uint4*>(&c[side]) = *reinterpret_cast<const uint4*>(src);
                s[side] = (side ? p.vs : p.ks)[row];
            }
        }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const RowsArg& o = side ? v : k;
        T* dst = static_cast<T*>(o.data) + (int64_t)t * o.ts + (int64_t)h * o.hs + part;
        float x[16];
        if (!has) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.0f;
        } else if constexpr (sizeof(C) > 1) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = to_f32(c[side].v[i]);
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(&c[side]);
            codes4(w.x, C{}, x);
            codes4(w.y, C{}, x + 4);
            codes4(w.z, C{}, x + 8);
            codes4(w.w, C{}, x + 12);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= s[side];
        }
        constexpr int V = 16 / sizeof(T);
        // a lane's 32 bytes as whole sectors, where the rows allow it
        const bool wide = ((reinterpret_cast<uintptr_t>(o.data) | (uintptr_t)(o.ts * sizeof(T)) | (uintptr_t)(o.hs * sizeof(T))) & 31) == 0;
        if (wide) {
#pragma unroll
            for (int i = 0; i < 16; i += 2 * V) {
                Raw32 r;
#pragma unroll
                for (int j = 0; j < 2 * V; j += 2) raw_put2<T>(r, j, x[i + j], x[i + j + 1]);
                store_raw32(dst + i, nullptr, r, true);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += V) store_f32<V>(dst + i, x + i);
        }
    }
}

}  // namespace xp
