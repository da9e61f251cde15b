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

// keys of a sequence: the end of its last tile or unit stays within 32 bits with a sign
constexpr uint64_t SERVE_MAX_KEYS = 0x7FFFFF00u;

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
    const int32_t lo = ld_now(a.starts + b), hi = ld_now(a.starts + b + 1);
    s.q0 = (uint32_t)min(max(lo, 0), (int32_t)a.tokens);
    s.nq = (uint32_t)max(min(max(hi, 0), (int32_t)a.tokens) - (int32_t)s.q0, 0);
    if (a.pages.k) {
        const uint64_t most = min((uint64_t)a.table_width << a.pages.page_shift, SERVE_MAX_KEYS);
        const int32_t n = max(ld_now(a.kv_lens + b), 0);
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

}  // namespace xp
