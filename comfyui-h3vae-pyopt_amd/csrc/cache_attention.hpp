// What the kernels of attention over the INT8 K/V cache share: their arguments, and how the keys of a tile of query rows
// are split and joined.
#pragma once

#include "h3v_paged.hpp"

namespace h3v {

constexpr float kLazy = 8.0f;         // log2 margin of the lazy softmax maximum
// log2 of the weight at the reference maximum.  Weights stay <= 2^(kLazy + kLift), within fp16, and those down to 2^-21 of
// the reference keep all their bits: many keys far below one that stands out lose nothing of their sum.  The sums carry the
// same factor, which the division takes out.
constexpr float kLift = 7.0f;
// References up to here: the exponent of a weight is one fma of score, factor and reference, which carries the product's bits that
// the reference, a rounded maximum, has lost, half a unit at most: weights stay within 2^15.5.  Beyond, where such
// bits would be whole powers of two, the product is rounded as the maximum was.
constexpr float kFar = 4194304.0f;
// Unnormalised outputs, in registers and in the workspace, are 2^-kOutDrop of what they stand for, which the last division takes
// back.  A bf16 value goes up to 2^128, and the sum of its weights (at most 2^15 each, 2^7 at the maximum) would pass fp32's
// range; with 2^-26 it may be 2^26, 2^19 keys at the maximum.  The least scale, 1e-30, stays a normal number.
constexpr int kOutDrop = 26;
constexpr float kInf = __builtin_inff();

struct AttnParams {
    Sequences s;
    const uint16_t* q;
    int64_t q_ts, q_hs;
    const int8_t *k, *v;
    const float *ks, *vs;
    float c;               // scale * log2(e)
    int causal, heads, kv_heads, group;
    uint16_t* o;           // [tokens][heads][D]
    int splits, slots;     // of this launch, and of the workspace
    float* part;           // [slots][tokens * heads][D] unnormalised outputs, then as many (maximum, sum) pairs
    const int* sel;        // [tokens][kv_heads][blocks] logical pages
    int blocks;
    int tile_rows;         // query rows ((token, head of the group) pairs of a kv head) of a tile
    int least;             // least pages of a split
    // Calls whose sequences differ run both kernels: sequences of at least this many rows of a kv head are for the long tiles,
    // which then find theirs by counting, the others for the 16-row tiles.  0: one kernel serves all of them.
    int long_rows;
};

__device__ __forceinline__ bool is_long(const AttnParams& p, const Span& sp) { return sp.n * p.group >= p.long_rows; }

// How a tile of rows shares its pages out: pages up to the last key that any of its rows sees, split into runs of
// `per` pages.
struct Split {
    int pages, per, active;
};

__device__ __forceinline__ Split split_pages(const AttnParams& p, int pages) {
    Split r;
    r.pages = pages;
    const int per = (pages + p.splits - 1) / p.splits;
    r.per = per > p.least ? per : p.least;
    r.active = (pages + r.per - 1) / r.per;
    return r;
}

// keys that new token i of the sequence sees
__device__ __forceinline__ int keys_seen(const AttnParams& p, const Span& sp, int i, int page) {
    const int64_t cap = (int64_t)p.s.width * page;
    int64_t n = p.causal ? (int64_t)sp.len - sp.n + i + 1 : sp.len;
    n = n < cap ? n : cap;
    return n > 0 ? (int)n : 0;
}

// a reference past kFar; a row without one, or with an infinite score, whose result is NaN, has none
__device__ __forceinline__ bool is_far(float reference) { return __builtin_fabsf(reference) > kFar && __builtin_fabsf(reference) < kInf; }

// merge weight of a part with reference maximum m under the common maximum top
__device__ __forceinline__ float part_weight(float m, float top) {
    return m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

// Launches the kernel of long row tiles (cache_prefill.hip); `rows` of a kv head in the largest sequence.
struct PrefillPlan {
    int tile_rows, splits, least;
};
// mixed: sequences that differ, whose rows only the packed tokens bound.
PrefillPlan plan_prefill(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t width, int64_t page,
                         int64_t dim, bool causal, bool mixed);
// Selected pages for tiles of several tokens (cache_selected.hip): tokens of a tile, 1 where the other kernel serves.
int selected_tile(int64_t tokens, int64_t batch, int64_t width, int64_t group, int64_t blocks);
int launch_selected(const char* what, const AttnParams& p, int tile, int dtype, int64_t dim, int64_t page, hipStream_t stream);
void launch_prefill(const AttnParams& p, int dtype, int64_t dim, int64_t page, int64_t rows, hipStream_t stream);

}  // namespace h3v
