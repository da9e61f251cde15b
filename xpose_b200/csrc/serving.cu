// Serving entry points of libxp_cuda.so: rotary rows, the paged cache and its
// attentions. A translation unit of its own, built beside xp_cuda.cu.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "host.cuh"
#include "serving_few.cuh"

using namespace xp;

namespace {

#define REQUIRE(cond, ...)                                      \
    do {                                                        \
        if (!(cond)) return fail(XP_ERR_INVALID, __VA_ARGS__);  \
    } while (0)

xp_status launched(const char* who, cudaError_t e) {
    if (e == cudaSuccess) return XP_OK;
    return fail(XP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

size_t bytes_of(uint32_t dtype) { return dtype == XP_F32 ? 4 : dtype == XP_F16 || dtype == XP_BF16 ? 2 : 1; }

// `align`: the elements every row has to be aligned to (a power of two)
xp_status check_rows(const char* who, const char* name, const xp_rows* r, uint32_t align) {
    REQUIRE(r, "%s: argument '%s' is null", who, name);
    REQUIRE(r->data || r->tokens == 0, "%s: '%s' has no data", who, name);
    REQUIRE(r->dtype <= XP_BF16, "%s: '%s' must be F32, F16 or BF16", who, name);
    REQUIRE(r->heads && r->dim, "%s: '%s' has no heads or no values in a head", who, name);
    REQUIRE(r->token_stride % align == 0 && r->head_stride % align == 0 &&
                (uintptr_t)r->data % (align * bytes_of(r->dtype)) == 0,
            "%s: the rows of '%s' must be aligned to %zu bytes", who, name, align * bytes_of(r->dtype));
    return XP_OK;
}
// Two of r's rows have an element in common: |dt ts + dh hs| < dim for some pair
// of distances that are not both zero.
bool rows_overlap(const xp_rows* r) {
    using wide = unsigned __int128;
    // a: the axis of fewer rows
    wide a = (wide)(r->head_stride < 0 ? -(__int128)r->head_stride : r->head_stride), na = r->heads;
    wide b = (wide)(r->token_stride < 0 ? -(__int128)r->token_stride : r->token_stride), nb = r->tokens;
    if (na > nb) {
        std::swap(a, b);
        std::swap(na, nb);
    }
    const wide dim = r->dim;
    if ((na > 1 && a < dim) || (nb > 1 && b < dim)) return true;
    if (na <= 1 || nb <= 1 || b >= (na - 1) * a + dim || a >= (nb - 1) * b + dim) return false;  // the usual layouts
    for (wide i = 1; i < na; ++i) {
        const wide j = i * a / b;  // the distances along the other axis that come nearest
        if ((j > 0 && j < nb && i * a - j * b < dim) || (j + 1 < nb && (j + 1) * b - i * a < dim)) return true;
    }
    return false;
}
xp_status check_written(const char* who, const char* name, const xp_rows* r) {
    REQUIRE(!rows_overlap(r), "%s: rows of '%s' overlap, and each is written", who, name);
    return XP_OK;
}
bool same_shape(const xp_rows* a, const xp_rows* b) {
    return a->tokens == b->tokens && a->heads == b->heads && a->dim == b->dim && a->dtype == b->dtype;
}
xp_status check_pages(const char* who, const xp_pages* p) {
    REQUIRE(p, "%s: argument 'pages' is null", who);
    REQUIRE(p->k && p->v, "%s: the pages have no data", who);
    REQUIRE(p->dtype >= XP_F16 && p->dtype <= XP_FP8_E4M3, "%s: pages must be F16, BF16, INT8 or FP8_E4M3", who);
    REQUIRE(p->page_size >= 8 && p->page_size <= 256 && !(p->page_size & (p->page_size - 1)),
            "%s: page_size must be a power of two from 8 to 256 (got %u)", who, p->page_size);
    REQUIRE(p->head_dim == 64 || p->head_dim == 128 || p->head_dim == 256,
            "%s: head_dim must be 64, 128 or 256 (got %u)", who, p->head_dim);
    REQUIRE(p->kv_heads && p->num_pages && p->num_pages < (1ull << 31) &&
                p->num_pages * p->page_size < 0xFFFFFFFFull / p->kv_heads,
            "%s: the pages are empty, or have 2^32 rows or more", who);
    REQUIRE(bytes_of(p->dtype) > 1 || (p->k_scale && p->v_scale), "%s: 8-bit pages need scales", who);
    REQUIRE((((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0 && (((uintptr_t)p->k_scale | (uintptr_t)p->v_scale) & 3) == 0,
            "%s: pages must be 16-byte aligned", who);
    return XP_OK;
}
xp_status check_rope(const char* who, const xp_rotary* r, uint32_t dim, uint32_t multiple) {
    REQUIRE(r->rot_dim && r->rot_dim <= dim && r->rot_dim % multiple == 0,
            "%s: rot_dim must be a multiple of %u up to %u (got %u)", who, multiple, dim, r->rot_dim);
    REQUIRE(r->layout <= XP_ROPE_INTERLEAVED, "%s: unknown rotary layout %u", who, r->layout);
    return XP_OK;
}
xp_status check_rope_data(const char* who, const xp_rotary* r) {
    REQUIRE(r->turns && r->positions, "%s: a rotation needs turns and positions", who);
    return XP_OK;
}
#define TRY(expr) \
    if (xp_status s_ = (expr); s_ != XP_OK) return s_

RowsArg rows_arg(const xp_rows* r, uint64_t t0 = 0) {
    return RowsArg{static_cast<char*>(r->data) + (int64_t)t0 * r->token_stride * (int64_t)bytes_of(r->dtype), r->token_stride,
                   r->head_stride};
}
RopeArg rope_arg(const xp_rotary* r) {
    if (!r) return RopeArg{};
    return RopeArg{reinterpret_cast<const unsigned long long*>(r->turns), r->positions, r->rot_dim,
                   r->layout == XP_ROPE_INTERLEAVED, r->magnitude, r->inverse ? -1.0f : 1.0f};
}
PagesArg pages_arg(const xp_pages* p) {
    return PagesArg{p->k, p->v, p->k_scale, p->v_scale, p->num_pages * p->page_size,
                    (uint32_t)__builtin_ctz(p->page_size), p->kv_heads};
}

// The driver's tensor map encoder (the library does not link libcuda).
PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return f;
}
// Rows as boxes of `width` bytes x rows, swizzled by that width. Packed:
// [tokens][heads][dim], rows along tokens; paged: [pages * heads][page][dim].
xp_status row_map(const char* who, CUtensorMap* m, CUtensorMapDataType type, uint32_t width, uint32_t size, void* data,
                  uint64_t dim, const uint64_t (&n)[2], const uint64_t (&stride)[2], const uint32_t (&box)[2]) {
    const auto encode = map_encoder();
    if (!encode) return fail(XP_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available", who);
    const cuuint64_t dims[3] = {dim, n[0], n[1]}, strides[2] = {stride[0], stride[1]};
    const cuuint32_t boxes[3] = {width / size, box[0], box[1]}, ones[3] = {1, 1, 1};
    const CUresult r = encode(m, type, 3, data, dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(XP_ERR_INVALID, "%s: the rows do not fit a tensor map (%d)", who, (int)r);
    return XP_OK;
}

// The attentions' scratch: the error word; the row tiles' parts
// (kinds, then sums); the few-row kernel's tickets and sums. The sums share
// their room: a call uses one kind.
constexpr size_t SCRATCH_HEADS = 256, SCRATCH_TICKETS = 8192, SCRATCH_TICKET_COUNT = 1024;
constexpr size_t SCRATCH_SLOTS = SCRATCH_TICKETS + SCRATCH_TICKET_COUNT * 4;
static_assert(SCRATCH_HEADS + 2 * AT_MAX_CTAS * 16 <= SCRATCH_TICKETS, "scratch");

template <class T, class C, int W>
xp_status launch_tiles(const char* who, const ServeAttnArgs& a, void* scratch, cudaStream_t st) {
    using G = AtCfg<T, C, W>;
    static_assert(G::smem <= 227 * 1024 && AT_MAX_BATCH * 4 <= G::row_off, "shared memory");
    static std::atomic<bool> attr_set[kMaxDevices];
    auto kernel = attn_tile_kernel<T, C, W>;
    if (cudaError_t e = smem_attr_once(attr_set, kernel, G::smem); e != cudaSuccess)
        return fail(XP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    const uint32_t ctas = std::min<uint32_t>((uint32_t)sm_count(), AT_MAX_CTAS);
    AtWork w{};
    w.slot_bytes = G::ROWS * (G::D * 4 + 8);
    w.heads = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(scratch) + SCRATCH_HEADS);
    w.slots = static_cast<unsigned char*>(scratch) + SCRATCH_SLOTS;
    static_assert(SCRATCH_SLOTS + 2ull * AT_MAX_CTAS * G::ROWS * (G::D * 4 + 8) <= XP_SERVING_SCRATCH_BYTES, "scratch");
    w.sub_tokens = 128 / a.group;
    w.tile_tokens = w.sub_tokens * G::NQ;
    w.least_units = 2;
    w.split_over = AT_COST + 1;
    CUtensorMap qm{}, km{}, vm{};
    const CUtensorMapDataType type =
        std::is_same_v<T, bf16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    {
        const uint64_t n[2] = {a.heads, a.tokens};
        const uint64_t stride[2] = {a.heads > 1 ? (uint64_t)a.q.hs * 2 : G::D * 2, a.tokens > 1 ? (uint64_t)a.q.ts * 2 : G::D * 2};
        const uint32_t box[2] = {a.group, w.sub_tokens};
        TRY(row_map(who, &qm, type, 128, 2, a.q.data, G::D, n, stride, box));
    }
    if constexpr (!G::Q8) {
        if (a.pages.k) {
            const uint32_t ps = 1u << a.pages.page_shift;
            const uint64_t n[2] = {ps, (a.pages.slots >> a.pages.page_shift) * a.kv_heads};
            const uint64_t stride[2] = {G::D * 2, (uint64_t)ps * G::D * 2};
            const uint32_t kbox[2] = {std::min<uint32_t>(ps, AT_KEYS), 1}, vbox[2] = {std::min<uint32_t>(ps, G::VKEYS), 1};
            TRY(row_map(who, &km, type, 128, 2, a.pages.k, G::D, n, stride, kbox));
            TRY(row_map(who, &vm, type, 128, 2, a.pages.v, G::D, n, stride, vbox));
        } else {
            // a lone head or token has no stride of its own; one head for all (stride 0) is a lone head
            w.head_step = 1;
            const uint32_t heads = a.kv_heads;
            for (const RowsArg* r : {&a.k, &a.v})
                if (heads > 1 && r->hs == 0) w.head_step = 0;
            const uint32_t mh = w.head_step ? heads : 1;
            const uint64_t n[2] = {mh, a.tokens};
            const uint32_t kbox[2] = {1, AT_KEYS}, vbox[2] = {1, G::VKEYS};
            const uint64_t ks[2] = {mh > 1 ? (uint64_t)a.k.hs * 2 : G::D * 2, a.tokens > 1 ? (uint64_t)a.k.ts * 2 : G::D * 2};
            const uint64_t vs[2] = {mh > 1 ? (uint64_t)a.v.hs * 2 : G::D * 2, a.tokens > 1 ? (uint64_t)a.v.ts * 2 : G::D * 2};
            TRY(row_map(who, &km, type, 128, 2, a.k.data, G::D, n, ks, kbox));
            TRY(row_map(who, &vm, type, 128, 2, a.v.data, G::D, n, vs, vbox));
        }
    }
    cudaError_t e = launch_ex(kernel, dim3(ctas), dim3(G::THREADS), G::smem, st, 1, true, a, w, qm, km, vm);
    if (e == cudaSuccess)
        e = launch_ex(attn_join_kernel<T, W, G::ROWS>, dim3(ctas, G::ROWS / 32 * W), dim3(256), 0, st, 1, true, a, w, ctas);
    if (e != cudaSuccess) return fail(XP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return XP_OK;
}

template <class T, class C, int W, int NR>
xp_status launch_few(const char* who, const ServeAttnArgs& a, void* scratch, cudaStream_t st) {
    using G = FwCfg<T, C, W, NR>;
    constexpr size_t slot_bytes = 8 * NR * (G::D * 4 + 8);
    static_assert(G::BYTES <= 227 * 1024, "shared memory");
    constexpr uint32_t most = 4 * AT_MAX_CTAS;
    static_assert(most <= SCRATCH_TICKET_COUNT && SCRATCH_SLOTS + 2 * most * slot_bytes <= XP_SERVING_SCRATCH_BYTES, "scratch");
    static std::atomic<bool> attr_set[kMaxDevices];
    auto kernel = attn_few_kernel<T, C, W, NR>;
    if (cudaError_t e = smem_attr_once(attr_set, kernel, G::smem); e != cudaSuccess)
        return fail(XP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    unsigned char* const s = static_cast<unsigned char*>(scratch);
    FwWork w{};
    w.tickets = reinterpret_cast<uint32_t*>(s + SCRATCH_TICKETS);
    w.slots = s + SCRATCH_SLOTS;
    w.slot_bytes = slot_bytes;
    CUtensorMap km, vm;
    const uint32_t ps = 1u << a.pages.page_shift;
    const uint64_t n[2] = {ps, (a.pages.slots >> a.pages.page_shift) * a.kv_heads};
    const uint64_t stride[2] = {G::RB, (uint64_t)ps * G::RB};
    const uint32_t box[2] = {std::min<uint32_t>(ps, G::KPS), 1};
    const CUtensorMapDataType type = G::Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : std::is_same_v<T, bf16> ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    TRY(row_map(who, &km, type, G::RB < 128 ? 64 : 128, sizeof(C), a.pages.k, G::D, n, stride, box));
    TRY(row_map(who, &vm, type, G::RB < 128 ? 64 : 128, sizeof(C), a.pages.v, G::D, n, stride, box));
    const uint32_t ctas = std::min<uint32_t>((uint32_t)sm_count() * G::CTAS, most);
    if (cudaError_t e = launch_ex(kernel, dim3(ctas), dim3(128), G::smem, st, 1, true, a, w, km, vm); e != cudaSuccess)
        return fail(XP_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return XP_OK;
}

// Calls f with a value of the type (and the W = dim / 64) that was asked for.
template <class F> xp_status for_type(uint32_t dtype, F f) {
    switch (dtype) {
        case XP_F32: return f(float{});
        case XP_F16: return f(__half{});
        default: return f(bf16{});
    }
}
template <class F> xp_status for_cache(uint32_t dtype, F f) {
    switch (dtype) {
        case XP_F16: return f(__half{});
        case XP_BF16: return f(bf16{});
        case XP_INT8: return f(int8c{});
        default: return f(fp8c{});
    }
}
template <class F> xp_status for_dim(uint32_t dim, F f) {
    switch (dim) {
        case 64: return f(std::integral_constant<int, 1>{});
        case 128: return f(std::integral_constant<int, 2>{});
        default: return f(std::integral_constant<int, 4>{});
    }
}

// f(first token, tokens, grid) for as many tokens at a time as keep a launch's
// thread numbers in 32 bits.
template <class F> xp_status in_parts(const char* who, uint64_t tokens, uint64_t per_token, uint32_t block, F f) {
    REQUIRE(per_token < (1ull << 31), "%s: too many values in a token", who);
    const uint64_t most = std::max<uint64_t>((1ull << 31) / per_token, 1);
    for (uint64_t t0 = 0; t0 < tokens; t0 += most) {
        const uint64_t n = std::min(tokens - t0, most);
        TRY(f(t0, (uint32_t)n, (unsigned)((n * per_token + block - 1) / block)));
    }
    return XP_OK;
}

}  // namespace

extern "C" {

xp_status xp_rope_turns(uint64_t* turns, float* magnitude, uint32_t rot_dim, double theta, uint32_t stretch,
                        double factor, double original, double slow, double fast) {
    const char* who = "rope_turns";
    REQUIRE(turns, "%s: argument 'turns' is null", who);
    REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0, "%s: rot_dim must be even (got %u)", who, rot_dim);
    REQUIRE(theta > 1.0 && std::isfinite(theta), "%s: theta must be above 1", who);
    REQUIRE(stretch <= XP_ROPE_PARTS, "%s: unknown stretch %u", who, stretch);
    REQUIRE(stretch == XP_ROPE_PLAIN || (factor >= 1.0 && std::isfinite(factor)), "%s: factor must be at least 1", who);
    REQUIRE(stretch != XP_ROPE_BASE || rot_dim > 2, "%s: a stretched base needs rot_dim above 2", who);
    REQUIRE(stretch != XP_ROPE_PARTS || (original > 0 && fast > slow), "%s: parts need original > 0 and fast > slow", who);
    const double two_pi = 6.283185307179586476925286766559;
    if (stretch == XP_ROPE_BASE) theta *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / rot_dim);
        if (stretch == XP_ROPE_LINEAR) f /= factor;
        if (stretch == XP_ROPE_PARTS) {
            const double g = std::fmin(1.0, std::fmax(0.0, (original * f / two_pi - slow) / (fast - slow)));
            f *= g + (1.0 - g) / factor;
        }
        turns[i] = (uint64_t)std::ldexp(f / two_pi, 64);  // f <= 1: below 2^62
    }
    if (magnitude) *magnitude = stretch == XP_ROPE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return XP_OK;
}

xp_status xp_rope_rows(void* stream, const xp_rows* out, const xp_rows* in, const xp_rotary* rope) {
    const char* who = "rope_rows";
    TRY(check_rows(who, "out", out, 1));
    TRY(check_rows(who, "in", in, 1));
    REQUIRE(rope, "%s: argument 'rope' is null", who);
    REQUIRE(same_shape(out, in), "%s: 'out' and 'in' differ in shape or type", who);
    TRY(check_rope(who, rope, in->dim, 2));
    TRY(check_written(who, "out", out));
    REQUIRE(out->data != in->data || in->tokens == 0 ||
                ((in->tokens == 1 || out->token_stride == in->token_stride) &&
                 (in->heads == 1 || out->head_stride == in->head_stride)),
            "%s: 'out' and 'in' share their data but not their strides", who);
    if (in->tokens == 0) return XP_OK;
    TRY(check_rope_data(who, rope));
    // vectors of 16 bytes where every row allows them, else one pair a thread
    const uint32_t vec = (uint32_t)(16 / bytes_of(in->dtype));
    bool wide = rope->rot_dim % (2 * vec) == 0 && in->dim % vec == 0;
    for (const xp_rows* r : {out, in})
        wide = wide && r->token_stride % vec == 0 && r->head_stride % vec == 0 && (uintptr_t)r->data % 16 == 0;
    const uint32_t vp = wide ? vec : 1;
    const uint32_t units = rope->rot_dim / 2 / vp + (in->dim - rope->rot_dim + 2 * vp - 1) / (2 * vp);
    // Heads a thread: enough to share the angles, as long as the GPU stays full.
    uint32_t hpt = 1;
    while (hpt < 8 && hpt < in->heads && (uint64_t)in->tokens * units * in->heads / (2 * hpt) >= (uint64_t)sm_count() * 2048)
        hpt *= 2;
    // 32-byte accesses where a unit's values lie side by side and every row allows it
    bool side = wide && in->dim % (2 * vec) == 0;
    for (const xp_rows* r : {out, in})
        side = side && r->token_stride % (2 * vec) == 0 && r->head_stride % (2 * vec) == 0 && (uintptr_t)r->data % 32 == 0;
    const bool copy = out->data != in->data;
    const uint64_t per_token = (uint64_t)((in->heads + hpt - 1) / hpt) * units;
    return in_parts(who, in->tokens, per_token, 256, [&](uint64_t t0, uint32_t n, unsigned grid) {
        return for_type(in->dtype, [&](auto t) {
            using T = decltype(t);
            auto k = wide ? rope_rows_kernel<T, 16 / sizeof(T)> : rope_rows_kernel<T, 1>;
            RopeArg r = rope_arg(rope);
            r.positions += t0;
            return launched(who, launch_ex(k, dim3(grid), dim3(256), 0, (cudaStream_t)stream, 1, true, rows_arg(out, t0),
                                           rows_arg(in, t0), r, n, in->heads, in->dim, hpt, units, copy, side));
        });
    });
}

xp_status xp_kv_write(void* stream, const xp_pages* pages, const xp_rows* k, const xp_rows* v, const int64_t* slots,
                      const xp_rotary* rope) {
    const char* who = "kv_write";
    TRY(check_pages(who, pages));
    TRY(check_rows(who, "k", k, 8));
    TRY(check_rows(who, "v", v, 8));
    REQUIRE(same_shape(k, v) && k->heads == pages->kv_heads && k->dim == pages->head_dim,
            "%s: 'k', 'v' and the pages differ in shape or type", who);
    if (rope) TRY(check_rope(who, rope, k->dim, 8));
    if (k->tokens == 0) return XP_OK;
    if (rope) TRY(check_rope_data(who, rope));
    REQUIRE(slots, "%s: argument 'slots' is null", who);
    return in_parts(who, k->tokens, (uint64_t)k->heads * (k->dim / 8), 256, [&](uint64_t t0, uint32_t n, unsigned grid) {
        return for_type(k->dtype, [&](auto t) {
            return for_cache(pages->dtype, [&](auto c) {
                return for_dim(k->dim, [&](auto d) {
                    RopeArg r = rope_arg(rope);
                    if (rope) r.positions += t0;
                    return launched(who, launch_ex(kv_write_kernel<decltype(t), decltype(c), d.value>, dim3(grid), dim3(256),
                                                   0, (cudaStream_t)stream, 1, true, pages_arg(pages), rows_arg(k, t0),
                                                   rows_arg(v, t0), slots + t0, n, r, rope != nullptr));
                });
            });
        });
    });
}

xp_status xp_kv_read(void* stream, const xp_pages* pages, const xp_rows* k, const xp_rows* v, const int64_t* slots) {
    const char* who = "kv_read";
    TRY(check_pages(who, pages));
    TRY(check_rows(who, "k", k, 1));
    TRY(check_rows(who, "v", v, 1));
    const uint32_t vec = (uint32_t)(16 / bytes_of(k->dtype));
    TRY(check_rows(who, "k", k, vec));
    TRY(check_rows(who, "v", v, vec));
    TRY(check_written(who, "k", k));
    TRY(check_written(who, "v", v));
    REQUIRE(same_shape(k, v) && k->heads == pages->kv_heads && k->dim == pages->head_dim,
            "%s: 'k', 'v' and the pages differ in shape or type", who);
    if (k->tokens == 0) return XP_OK;
    REQUIRE(slots, "%s: argument 'slots' is null", who);
    return in_parts(who, k->tokens, (uint64_t)k->heads * (k->dim / 16), 256, [&](uint64_t t0, uint32_t n, unsigned grid) {
        return for_type(k->dtype, [&](auto t) {
            return for_cache(pages->dtype, [&](auto c) {
                return for_dim(k->dim, [&](auto d) {
                    return launched(who, launch_ex(kv_read_kernel<decltype(t), decltype(c), d.value>, dim3(grid), dim3(256),
                                                   0, (cudaStream_t)stream, 1, true, pages_arg(pages), rows_arg(k, t0),
                                                   rows_arg(v, t0), slots + t0, n));
                });
            });
        });
    });
}

}  // extern "C"

namespace {

xp_status attention(const char* who, void* stream, const xp_rows* out, const xp_rows* q, const xp_rows* k,
                    const xp_rows* v, const xp_pages* pages, const int32_t* table, uint32_t table_width,
                    const int32_t* kv_lens, const int32_t* starts, uint32_t batch, uint32_t q_most, uint32_t window,
                    float scale, float* lse, void* scratch) {
    TRY(check_rows(who, "q", q, 8));
    TRY(check_rows(who, "out", out, 8));
    REQUIRE(q->dtype != XP_F32, "%s: 'q' must be F16 or BF16", who);
    REQUIRE((q->token_stride > 0 || q->tokens <= 1) && (q->head_stride > 0 || q->heads <= 1) && q->token_stride >= 0 &&
                q->head_stride >= 0,
            "%s: 'q' needs positive strides", who);
    REQUIRE(same_shape(q, out), "%s: 'q' and 'out' differ in shape or type", who);
    TRY(check_written(who, "out", out));
    REQUIRE(q->dim == 64 || q->dim == 128 || q->dim == 256, "%s: dim must be 64, 128 or 256 (got %u)", who, q->dim);
    uint32_t kv_heads, cache;
    if (pages) {
        TRY(check_pages(who, pages));
        REQUIRE(pages->head_dim == q->dim, "%s: 'q' and the pages differ in dim", who);
        REQUIRE(bytes_of(pages->dtype) == 1 || pages->dtype == q->dtype, "%s: 16-bit pages must have q's type", who);
        kv_heads = pages->kv_heads;
        cache = pages->dtype;
    } else {
        TRY(check_rows(who, "k", k, 8));
        TRY(check_rows(who, "v", v, 8));
        for (const xp_rows* r : {k, v})
            REQUIRE(r->token_stride >= 0 && r->head_stride >= 0 && (r->token_stride > 0 || r->tokens <= 1),
                    "%s: 'k' and 'v' need strides that are not negative, and a token stride", who);
        REQUIRE((k->head_stride == 0) == (v->head_stride == 0) || k->heads <= 1,
                "%s: one of 'k' and 'v' has one head for all, the other not", who);
        REQUIRE(same_shape(k, v) && k->tokens == q->tokens && k->dim == q->dim && k->dtype == q->dtype,
                "%s: 'q', 'k' and 'v' differ in shape or type", who);
        kv_heads = k->heads;
        cache = q->dtype;
    }
    REQUIRE(q->heads % kv_heads == 0, "%s: %u heads are no multiple of %u kv heads", who, q->heads, kv_heads);
    REQUIRE(q->heads / kv_heads <= 128, "%s: more than 128 heads share a kv head", who);
    REQUIRE(batch <= AT_MAX_BATCH, "%s: at most %u sequences a call", who, AT_MAX_BATCH);
    REQUIRE(q->tokens <= 0x7FFFFFFFu, "%s: too many tokens", who);
    REQUIRE(std::isfinite(scale) && scale >= 0.0f, "%s: scale must be finite and not negative", who);
    if (q->tokens == 0) return XP_OK;
    REQUIRE(starts, "%s: argument 'starts' is null", who);
    REQUIRE(scratch && (uintptr_t)scratch % 16 == 0, "%s: 'scratch' must be 16-byte aligned", who);
    if (pages) {
        REQUIRE(kv_lens, "%s: argument 'kv_lens' is null", who);
        REQUIRE(table || table_width == 0, "%s: argument 'table' is null", who);
        REQUIRE(((uint64_t)table_width * pages->page_size) < (1ull << 31), "%s: table rows of 2^31 keys or more", who);
    }
    ServeAttnArgs a{};
    a.out = rows_arg(out);
    a.q = rows_arg(q);
    if (pages) {
        a.pages = pages_arg(pages);
    } else {
        a.k = rows_arg(k);
        a.v = rows_arg(v);
    }
    a.table = table;
    a.table_width = table_width;
    a.kv_lens = kv_lens;
    a.starts = starts;
    a.batch = batch;
    a.tokens = q->tokens;
    a.heads = q->heads;
    a.kv_heads = kv_heads;
    a.group = q->heads / kv_heads;
    a.q_most = q_most;
    a.window = window;
    a.scale_log2 = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)q->dim)) * 1.4426950408889634f;
    a.lse = lse;
    a.err = static_cast<uint32_t*>(scratch) + 1;
    return for_type(q->dtype, [&](auto t) {
        return for_cache(cache, [&](auto c) {
            return for_dim(q->dim, [&](auto d) {
                using T = decltype(t);
                using C = decltype(c);
                if constexpr (sizeof(T) == 2 && (sizeof(C) == 1 || std::is_same_v<C, T>)) {
                    // Up to 16 rows a kv head: read-bound, one pass of warp products. Measured on both
                    // kernels, us, 64 sequences of 4096 keys, few-row / tile: 32 / 8 heads of 128, e4m3,
                    // 4 rows 116 / 404, 16 rows 140 / 406; 16 / 4 of 64, bf16, 16 rows 58 / 116; 4 / 1 of
                    // 256, e4m3, 8 rows 45 / 74. What this rule does not serve: 256-wide heads with 16
                    // rows, bf16 86 / 61, int8 88 / 75, e4m3 87 / 74
                    const uint64_t rows = (uint64_t)q_most * a.group;
                    if (pages && rows <= 8) return launch_few<T, C, d.value, 1>(who, a, scratch, (cudaStream_t)stream);
                    if (pages && rows <= 16) return launch_few<T, C, d.value, 2>(who, a, scratch, (cudaStream_t)stream);
                    return launch_tiles<T, C, d.value>(who, a, scratch, (cudaStream_t)stream);
                } else {
                    return fail(XP_ERR_UNSUPPORTED, "%s: no kernel for these types", who);
                }
            });
        });
    });
}

}  // namespace

extern "C" {

xp_status xp_attention_packed(void* stream, const xp_rows* out, const xp_rows* q, const xp_rows* k, const xp_rows* v,
                              const int32_t* starts, uint32_t batch, uint32_t window, float scale, float* lse,
                              void* scratch) {
    return attention("attention_packed", stream, out, q, k, v, nullptr, nullptr, 0, nullptr, starts, batch, 0, window,
                     scale, lse, scratch);
}

xp_status xp_attention_paged(void* stream, const xp_rows* out, const xp_rows* q, const xp_pages* pages,
                             const int32_t* table, uint32_t table_width, const int32_t* kv_lens,
                             const int32_t* starts, uint32_t batch, uint32_t q_most, uint32_t window, float scale,
                             float* lse, void* scratch) {
    REQUIRE(pages, "attention_paged: argument 'pages' is null");
    return attention("attention_paged", stream, out, q, nullptr, nullptr, pages, table, table_width, kv_lens, starts,
                     batch, q_most, window, scale, lse, scratch);
}

}  // extern "C"
