// Attention of new tokens over the INT8 K/V cache (layout and lookups: h3v_paged.hpp):
//
//   o[t, h] = sum_j softmax_j(scale * q[t, h] . K[j]) V[j],   K[j] = s_k * code, V[j] = s_v * code
//
// over the keys j < len of the token's sequence (causal: up to the token's own position), or over the pages that
// a list names for every token and kv head.  A row without a key is zeros.  Query head h reads kv head h / G.
//
// One wave works on 16 query rows of one kv head ((token, head of the group) pairs) and KT keys at a time, all in
// registers: the products run on v_mfma_f32_16x16x32_f16 with the codes as exact fp16 integers.
//
//   S = K . Q^T    A = K rows: lane l reads 16 codes of one key, B = Q (fragments loaded once).  The order of the 32
//                  slots of a product is free as long as A and B agree, so a lane's 16 consecutive codes feed two
//                  products, and the key that row r of tile t stands for is free too: 16 (r / 4) + 4 t + r % 4 (64
//                  keys), so that lane group g = l / 16 ends up with the scores of 16 consecutive keys.
//   O^T += s_v (V^T . P^T)   A = V^T rows: lane l reads the codes of its group's consecutive keys of one dim, B = P, the
//                  scores of the same keys, already in place: no exchange between lanes and no LDS.
//
// The page's key scale joins the exponent's factor, its value scale multiplies the product of the page in fp32, so that
// the products see exact integers and fp16 weights.  The softmax keeps a lazy reference maximum: it moves only
// when a score passes it by 2^8, and the weights are 2^7 times those of the textbook, so that fp16 holds them down to 2^-21 with all
// bits.  fp32 sums and statistics; the row sums add the fp16
// weights that the product uses.  bf16 queries are scaled to at most 1 by a power of two, which the factor takes back.
//
// Single tokens are bound by memory: 64 sequences of up to 8001 tokens, 8 kv heads of 128, 778 MB of pages in 141 us, 5.5 TB/s
// (vector units 32%, matrix units 8%); two of up to 131071, 4 kv heads of 128, 227 MB in 51 us and 5 us for the join of 32 splits.
#include <algorithm>

#include "cache_rows.hpp"

namespace h3v {
namespace {

constexpr int kNW = 4;                // waves of a workgroup; they share out the pages of a split
constexpr int kNT = 64 * kNW;

// STREAM: a call of one row tile per kv head, whose pages are read once (8 kv heads of 128, pages of 64: 64 sequences of up to
// 8001 tokens 155 -> 141 us, 32 of 4000 48.6 -> 44.2, 8 of 2000 15.5 -> 14.3, one of 517 with 32 heads of 64 the same).
// Not for pages of 128 tokens, where a step reads half of each line of the values and the next one the other half
// (two sequences of 131071 tokens: 56 us without, 60 us with), nor for selected pages, which other tokens read too
// (16 tokens of 65000, 32 pages each, with the selection: 35.2 us without, 36.4 with; 2048 of one sequence: 143, 159).
// MIXED: not the sequences that are long (AttnParams::long_rows).  Tiles behind a sequence's first are mostly not there: they
// come last, so that their workgroups do not stand between those that have work.
template <int DT, int D, int P, bool SEL, bool STREAM, bool MIXED>
__global__ __launch_bounds__(kNT, 2) void cache_attention_kernel(AttnParams p) {
    using Tile = RowTile<DT, D, P>;
    __shared__ __attribute__((aligned(16))) Joined<D, kNW> joined;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15;

    int b, kvh, sp_i, tile, tiles;
    Span span;
    int64_t token = 0;
    int listed = -1;
    if constexpr (SEL) {
        token = blockIdx.x;
        kvh = blockIdx.y;
        sp_i = blockIdx.z;
        // the list does not wait for the sequence: its entries of the wave's first 64 pages
        const Split sp = split_pages(p, p.blocks);
        const int at = sp_i * sp.per + wave + lane * kNW;
        if (at < min(sp.pages, (sp_i + 1) * sp.per)) listed = p.sel[(token * p.kv_heads + kvh) * p.blocks + at];
        b = __builtin_amdgcn_readfirstlane(sequence_of(p.s, token));
        if (b < 0) {
            if (sp_i == 0)
                for (int e = tid; e < p.group * (D / 8); e += kNT)
                    *reinterpret_cast<u32x4*>(p.o + (token * p.heads + kvh * p.group) * D + 8 * e) = u32x4{0, 0, 0, 0};
            return;
        }
        span = span_of(p.s, b);
        tile = 0;
        tiles = 1;
    } else {
        sp_i = MIXED ? blockIdx.x % p.splits : blockIdx.x;
        kvh = blockIdx.y % p.kv_heads;
        tile = MIXED ? blockIdx.z : blockIdx.y / p.kv_heads;
        b = MIXED ? blockIdx.x / p.splits : blockIdx.z;
        if (b == p.s.batch) {   // rows of no sequence: zeros
            const int tiles = MIXED ? gridDim.z : gridDim.y / p.kv_heads;
            const int64_t lo = p.s.starts[0], hi = p.s.starts[p.s.batch], step = (int64_t)p.splits * p.kv_heads * tiles * kNT;
            const int64_t row = p.heads * (D / 8);
            for (int64_t e = (((int64_t)tile * p.kv_heads + kvh) * p.splits + sp_i) * kNT + tid; e < p.s.tokens * row; e += step) {
                const int64_t t = e / row;
                if (t < lo || t >= hi) *reinterpret_cast<u32x4*>(p.o + 8 * e) = u32x4{0, 0, 0, 0};
            }
            return;
        }
        span = span_of(p.s, b);
        if (MIXED && is_long(p, span)) return;
        tiles = (int)(((int64_t)span.n * p.group + 15) / 16);
    }
    const int tile_step = SEL ? 1 : (MIXED ? gridDim.z : gridDim.y / p.kv_heads);
    for (; tile < tiles; tile += tile_step) {
        // this lane's row: token i of the sequence, head
        int rows, i, head, seen, last;
        if constexpr (SEL) {
            rows = p.group;
            i = (int)(token - span.row);
            head = kvh * p.group + (col < rows ? col : 0);
            seen = keys_seen(p, span, i, P);
            last = seen;
        } else {
            const int r0 = tile * 16, all = span.n * p.group;
            rows = all - r0 < 16 ? all - r0 : 16;
            const int r = r0 + (col < rows ? col : 0);
            i = r / p.group;
            head = kvh * p.group + r % p.group;
            seen = keys_seen(p, span, i, P);
            last = keys_seen(p, span, (r0 + rows - 1) / p.group, P);
        }
        const int64_t trow = SEL ? token : span.row + i;
        const Split sp = split_pages(p, SEL ? p.blocks : (last + P - 1) / P);
        if (sp_i > 0 && sp_i >= sp.active) continue;
        const int j0 = sp_i * sp.per, j1 = min(sp.pages, j0 + sp.per);

        Tile rt;
        rt.load_rows(p.q + trow * p.q_ts + head * p.q_hs);
        rt.reset();
        // the wave's pages j0 + wave, + kNW, ...: up to 64 at a time, their ids and scales one per lane
        int my_id, my_j;
        float my_ks, my_vs;
        auto fetch = [&](int jb) {
            my_id = -1;
            my_j = 0;
            my_ks = my_vs = 0.0f;
            if (lane < min(64, (j1 - jb + kNW - 1) / kNW)) {
                my_j = jb + lane * kNW;
                if constexpr (SEL) my_j = jb == j0 + wave ? listed : p.sel[(token * p.kv_heads + kvh) * p.blocks + my_j];
                my_id = my_j >= 0 && my_j <= (last - 1) / P && last > 0 ? page_id(p.s, b, my_j) : -1;
            }
            if (my_id >= 0) {
                my_ks = p.ks[(int64_t)my_id * p.kv_heads + kvh];
                my_vs = p.vs[(int64_t)my_id * p.kv_heads + kvh] * (1.0f / (1 << kOutDrop));
            }
        };
        fetch(j0 + wave);
        rt.set_rows(p.c);
        for (int jb = j0 + wave; jb < j1; jb += 64 * kNW) {
            if (jb != j0 + wave) fetch(jb);
            const uint64_t there = __ballot(my_id >= 0);
            // pages that are not there are passed over: step u is the part u % NSUB of the (u / NSUB)-th one that is
            struct Step {
                typename Tile::Codes codes;
                int lane, sub;
            };
            uint64_t left = there;
            int sub = 0;
            Tile::template run<Step>(
                __popcll(there) * Tile::NSUB,
                [&](Step& w) {
                    w.lane = __builtin_ctzll(left);
                    w.sub = sub;
                    const int id = __builtin_amdgcn_readlane(my_id, w.lane);
                    rt.template load<STREAM>(w.codes, p.k, p.v, (int64_t)id * p.kv_heads + kvh, sub);
                    if (++sub == Tile::NSUB) {
                        sub = 0;
                        left &= left - 1;
                    }
                },
                [&](Step& w) {
                    const int key0 = __builtin_amdgcn_readlane(my_j, w.lane) * P + w.sub * Tile::KT;
                    if (Tile::NSUB > 1 && key0 >= last) return;
                    rt.attend(w.codes, key0, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_ks), w.lane)),
                              __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_vs), w.lane)), seen);
                });
        }

        // the waves' parts
        __syncthreads();   // the last tile's parts are read
        joined.put(rt, wave);
        __syncthreads();
        for (int e = tid; e < rows * (D / 4); e += kNT) {
            const int r = e / (D / 4), d = e % (D / 4) * 4;
            float top, sum;
            const f32x4 out = joined.get(r, d, top, sum);
            int64_t row;
            if constexpr (SEL) row = token * p.heads + kvh * p.group + r;
            else row = (span.row + (tile * 16 + r) / p.group) * p.heads + kvh * p.group + (tile * 16 + r) % p.group;
            if (sp.active > 1) {
                const int64_t at = (int64_t)sp_i * p.s.tokens * p.heads + row;
                *reinterpret_cast<f32x4*>(p.part + at * D + d) = out;
                if (d == 0) {
                    float* const pml = p.part + (int64_t)p.slots * p.s.tokens * p.heads * D + 2 * at;
                    pml[0] = top;
                    pml[1] = sum;
                }
            } else {
                put_row<DT>(p.o + row * D + d, out, row_inverse(top, sum));
            }
        }
    }
}

// Joins the splits of a tile's rows: parts rescaled to their largest reference maximum and added, in an order that is
// fixed.  WR waves per row (1, or all 4 where a row has many splits): lanes of 4 dims each, the others side by side.
// SEL: selected pages, a token to a workgroup; FLAT: the sequences that are long of a call of both kinds, a row to a wave by
// the packed tokens.
template <int DT, int D, int P, bool SEL, bool FLAT, int WR>
__global__ __launch_bounds__(256) void cache_attention_merge(AttnParams p) {
    constexpr int LD = D / 4, NP = 64 / LD * WR;     // lanes of a part, parts that run side by side
    __shared__ __attribute__((aligned(16))) float sums[WR > 1 ? WR : 1][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int d = lane % LD * 4, part = lane / LD + (WR > 1 ? wave * (64 / LD) : 0);
    int b, r, rows;
    const int kvh = blockIdx.y;
    Span span;
    int64_t token = 0;
    if constexpr (SEL) {
        token = blockIdx.x;
        b = __builtin_amdgcn_readfirstlane(sequence_of(p.s, token));
        if (b < 0) return;
        span = span_of(p.s, b);
        rows = p.group;
        r = WR > 1 ? 0 : wave;
    } else if constexpr (FLAT) {
        const int64_t at = (int64_t)blockIdx.x * 4 + wave;
        token = at / p.group;
        b = token < p.s.tokens ? __builtin_amdgcn_readfirstlane(sequence_of(p.s, token)) : -1;
        if (b < 0) return;
        span = span_of(p.s, b);
        if (!is_long(p, span)) return;
        rows = span.n * p.group;
        r = (int)(token - span.row) * p.group + (int)(at % p.group);
    } else {
        b = blockIdx.z;
        span = span_of(p.s, b);
        rows = p.long_rows > 0 && is_long(p, span) ? 0 : span.n * p.group;
        r = WR > 1 ? blockIdx.x : blockIdx.x * 4 + wave;
    }
    const int64_t stride = p.s.tokens * p.heads;
    const float* const pml = p.part + p.slots * stride * D;
    for (; r < rows; r += FLAT ? rows : (SEL ? 1 : gridDim.x) * (4 / WR)) {
        int pages = p.blocks;
        int64_t row;
        if constexpr (SEL) {
            row = token * p.heads + kvh * p.group + r;
        } else {
            const int end = min(rows, (r / p.tile_rows + 1) * p.tile_rows);
            pages = (keys_seen(p, span, (end - 1) / p.group, P) + P - 1) / P;
            row = (span.row + r / p.group) * p.heads + kvh * p.group + r % p.group;
        }
        const int active = split_pages(p, pages).active;
        if (active <= 1) continue;
        // at most 32 splits: one per lane
        const float2 mine = lane < active ? *reinterpret_cast<const float2*>(pml + 2 * (lane * stride + row)) : make_float2(-kInf, 0.0f);
        float top = mine.x;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off, 64));
        const float f = part_weight(mine.x, top);
        float sum = f * mine.y;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
        const float* const src = p.part + row * D + d;
#pragma unroll 8
        for (int s0 = 0; s0 < active; s0 += NP) {
            const int s = s0 + part;
            const float w = __shfl(f, s & 63, 64);
            const f32x4 v = *reinterpret_cast<const f32x4*>(src + (s < active ? s : 0) * stride * D);
#pragma unroll
            for (int x = 0; x < 4; ++x) out[x] = s < active ? __builtin_fmaf(w, v[x], out[x]) : out[x];
        }
#pragma unroll
        for (int off = LD; off < 64; off <<= 1)
#pragma unroll
            for (int x = 0; x < 4; ++x) out[x] += __shfl_xor(out[x], off, 64);
        if constexpr (WR > 1) {
            __syncthreads();   // the last row's sums are read
            if (lane < LD) *reinterpret_cast<f32x4*>(&sums[wave][d]) = out;
            __syncthreads();
            if (wave > 0) continue;
#pragma unroll
            for (int w = 1; w < WR; ++w) out += *reinterpret_cast<const f32x4*>(&sums[w][d]);
        }
        if (lane < LD) put_row<DT>(p.o + row * D + d, out, row_inverse(top, sum));
    }
}

// More splits than kWideSplits: a workgroup per row.
constexpr int kWideSplits = 8;

constexpr int kSplitPages = 4;

// Splits of the keys: about two workgroups for each CU, the most that it holds, of at least four pages, where there are 16; of
// at least 16 pages where one split has a workgroup for each CU already; at most 32, whose join is cheap.  us with one split / for
// 256 workgroups / for 512, ragged batches of one token over up to that many, 8 kv heads of 128, pages of 64: 3 x 4000 35.5 / 16.7 /
// 15.5, 6 x 8000 61.5 / 32.8 / 27.4, 12 x 8000 64.3 / 50.4 / 39.4, 16 x 30000 - / 146 / 140, 48 x 4000 71 / 71 / 63.5, 63 x 4000, of
// one length, 87 / 87 / 94;  32 kv heads of 64: 12 x 2000 19.5 / 19.3 / 20.9;  1 x 16000 with 32 splits 16.0, with 64 18.2.
int plan_splits(int64_t units, int64_t pages) {
    if (pages < 16) return 1;
    const int64_t want = (512 + units * 2 / 3) / units, cap = pages / (units < 256 ? kSplitPages : 16);
    const int64_t splits = std::min<int64_t>({want, cap, 32});
    return splits > 1 ? (int)splits : 1;
}

// Selected pages are few: a workgroup for each CU (us for 256 / 512 workgroups, with the selection, 8 kv heads of 128: 4 tokens, 48
// pages each 26.3 / 29.6; 24, 32 pages 35.9 / 37.1).
int selected_splits(int64_t tokens, int64_t kv_heads, int64_t blocks) {
    const int64_t units = tokens * kv_heads;
    return blocks < 16 ? 1 : (int)std::min<int64_t>({(256 + units - 1) / units, blocks / kSplitPages, 32});
}

constexpr int64_t kMaxTokens = 1 << 24;

int64_t tiles_of(int64_t max_new, int64_t group) { return (max_new * group + 15) / 16; }

// Rows of a kv head in the largest sequence from which the long tiles of cache_prefill.hip serve.  Below, 16-row tiles read a
// sequence's pages few times; above, a row costs the long tiles less, at dim 128 earlier where (sequence, kv head) pairs alone
// fill the chip (us, 16-row / long tiles; batch x length, 8 kv heads): dim 128, 64 rows: 8 x 4000 36 / 37, 32 x 1000 34 / 31;
// 96 rows: 52 / 38, 45 / 34; dim 64, 128 rows: 24 / 31, 28 / 25; 256 rows: 43 / 42, 45 / 38; 32 kv heads, 56 rows, dim 128:
// 31 x 58 44 / 30, 31 x 300 53 / 50, dim 64: 24 / 29, 29 / 54.
int64_t prefill_rows(int64_t pairs, int64_t dim) { return dim == 64 ? 145 : (pairs >= 256 ? 49 : 81); }

constexpr int64_t kMaxWorkspace = 1 << 26;   // floats

// One kernel for all sequences, or the long tiles for those of at least long_rows rows and the 16-row tiles for the others:
// a call may bring a prompt and many single tokens, of which each kernel does only one kind well (8 kv heads of 128, four heads
// each; us, both / long tiles alone: 2048 new tokens and 63 single ones over 4000 178 / 380; 300 new and 15 single ones over 30000 194 / 441).
struct Plan {
    bool prefill;
    int tile_rows, splits, least, short_splits, long_rows, slots;
};

Plan plan_attention(int64_t tokens, int64_t batch, int64_t width, int64_t heads, int64_t kv_heads, int64_t dim, int64_t max_new,
                    bool causal, int64_t page) {
    const int64_t rows = max_new * (heads / kv_heads), least = prefill_rows(batch * kv_heads, dim);
    Plan plan = {false, 16, 1, kSplitPages, 1, 0, 1};
    if (rows >= least) {
        const bool mixed = max_new * batch > tokens;
        const PrefillPlan r = plan_prefill(tokens, batch, heads, kv_heads, rows, width, page, dim, causal, mixed);
        plan = {true, r.tile_rows, r.splits, r.least, mixed ? plan_splits(batch * kv_heads, width) : 1, mixed ? (int)least : 0, 1};
    } else {
        plan.splits = plan_splits(batch * kv_heads * tiles_of(max_new, heads / kv_heads), width);
    }
    // splits are for calls of few rows; a max_new far below the truth must not make a workspace of many
    while (plan.splits > 1 && plan.splits * tokens * heads * (dim + 2) > kMaxWorkspace) plan.splits /= 2;
    while (plan.short_splits > 1 && plan.short_splits * tokens * heads * (dim + 2) > kMaxWorkspace) plan.short_splits /= 2;
    plan.slots = plan.splits > plan.short_splits ? plan.splits : plan.short_splits;
    return plan;
}

int64_t ws_floats(int splits, int64_t tokens, int64_t heads, int64_t dim) {
    return splits > 1 ? splits * tokens * heads * (dim + 2) : 0;
}

int check(const char* what, int dtype, const AttnParams& p, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page, float scale) {
    const int rc = check_paged(what, dtype, p.s, kv_heads, dim, page);
    if (rc) return rc;
    H3V_REQUIRE(p.q && p.s.starts && p.k && p.v && p.ks && p.vs && p.o, "%s: null pointer argument", what);
    H3V_REQUIRE(p.s.tokens > 0 && p.s.tokens <= kMaxTokens, "%s: tokens must be in [1, 2^24]", what);
    H3V_REQUIRE(heads > 0 && heads <= 4096 && heads % kv_heads == 0, "%s: heads must be a multiple of the kv heads, up to 4096", what);
    H3V_REQUIRE(p.s.tokens * heads <= (1 << 30), "%s: tokens x heads must be at most 2^30", what);
    H3V_REQUIRE(p.q_ts > 0 && p.q_ts % 8 == 0 && p.q_hs > 0 && p.q_hs % 8 == 0,
                "%s: token/head strides must be positive multiples of 8 elements (16-byte rows)", what);
    H3V_REQUIRE(aligned(p.q, 16) && aligned(p.k, 16) && aligned(p.v, 16) && aligned(p.o, 16),
                "%s: q, the cache and the output must be 16-byte aligned", what);
    H3V_REQUIRE(aligned(p.ks, 4) && aligned(p.vs, 4), "%s: scales must be 4-byte aligned", what);
    H3V_REQUIRE(scale > 0.0f && scale < 1e30f, "%s: scale must be positive and finite", what);
    return H3V_OK;
}

}  // namespace
}  // namespace h3v

using namespace h3v;

extern "C" {

int64_t h3v_cache_attention_workspace_floats(int64_t tokens, int64_t batch, int64_t width, int64_t heads, int64_t kv_heads,
                                             int64_t dim, int64_t page, int causal, int64_t max_new) {
    if (tokens <= 0 || batch <= 0 || width <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || page <= 0 ||
        max_new <= 0)
        return -1;
    return ws_floats(plan_attention(tokens, batch, width, heads, kv_heads, dim, max_new, causal != 0, page).slots, tokens, heads, dim);
}

int h3v_cache_attention(int dtype, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                        const int* starts, const int* lens, const int* table, int64_t batch, int64_t width, int64_t heads,
                        int64_t kv_heads, int64_t dim, int64_t page, int64_t pages, const int8_t* k_cache,
                        const int8_t* v_cache, const float* k_scale, const float* v_scale, float scale, int causal,
                        int64_t max_new, uint16_t* out, float* workspace, int64_t workspace_floats, hipStream_t stream) {
    const char* what = "h3v_cache_attention";
    H3V_REQUIRE(batch > 0 && batch <= 32768 && width > 0 && width <= (1 << 23), "%s: batch or table width out of range", what);
    H3V_REQUIRE(kv_heads > 0, "%s: kv heads must be positive", what);
    AttnParams p = {{starts, lens, table, (int)batch, (int)width, tokens, pages}, q, q_token_stride, q_head_stride, k_cache,
                    v_cache, k_scale, v_scale, scale * 1.4426950408889634f, causal != 0, (int)heads, (int)kv_heads,
                    (int)(heads / kv_heads), out, 1, 1, workspace, nullptr, 0, 16, kSplitPages, 0};
    const int rc = check(what, dtype, p, heads, kv_heads, dim, page, scale);
    if (rc) return rc;
    H3V_REQUIRE(max_new > 0 && max_new <= tokens, "%s: max_new must be in [1, tokens]", what);
    const Plan plan = plan_attention(tokens, batch, width, heads, kv_heads, dim, max_new, causal != 0, page);
    p.slots = plan.slots;
    p.long_rows = plan.long_rows;
    const int64_t floats = ws_floats(p.slots, tokens, heads, dim);
    H3V_REQUIRE(floats == 0 || (workspace && workspace_floats >= floats && aligned(workspace, 16)),
                "%s: needs a 16-byte aligned workspace of %lld floats", what, (long long)floats);
    // workgroups stride over a sequence's row tiles, so max_new only sets how many there are
    int64_t rows = max_new * p.group;
    if (plan.prefill) {
        p.splits = plan.splits;
        p.tile_rows = plan.tile_rows;
        p.least = plan.least;
        // the packed rows' tiles, and one that is not full of every sequence that can be long; of those no more than fill
        // the chip, since most are not there (workgroups stride)
        const int64_t all = tokens * p.group, parts = std::min({batch, all / std::max(plan.long_rows, 1), (256 + kv_heads - 1) / kv_heads});
        if (plan.long_rows) rows = (all / p.tile_rows + parts) * p.tile_rows;
        if (rows > 0) launch_prefill(p, dtype, dim, page, rows, stream);
        if (plan.long_rows && p.splits > 1) {
            const dim3 merge((unsigned)((all + 3) / 4), (unsigned)kv_heads);
            by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
                hipLaunchKernelGGL((cache_attention_merge<dt(), d(), pg(), false, true, 1>), merge, dim3(256), 0, stream, p);
            });
        }
    }
    if (!plan.prefill || plan.long_rows) {
        p.splits = plan.long_rows ? plan.short_splits : plan.splits;
        p.tile_rows = 16;
        p.least = kSplitPages;
        if (plan.long_rows) rows = plan.long_rows - 1;
        const int64_t tiles = (rows + 15) / 16;   // at most 9: see prefill_rows; 65535 workgroups of y hold them
        const dim3 grid((unsigned)p.splits, (unsigned)(tiles * kv_heads), (unsigned)(batch + 1));
        const dim3 several((unsigned)(p.splits * (batch + 1)), (unsigned)kv_heads, (unsigned)tiles);
        by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
            constexpr bool kStream = pg() < 128;
            if (plan.long_rows) hipLaunchKernelGGL((cache_attention_kernel<dt(), d(), pg(), false, kStream, true>), several, dim3(kNT), 0, stream, p);
            else if (kStream && tiles == 1) hipLaunchKernelGGL((cache_attention_kernel<dt(), d(), pg(), false, kStream, false>), grid, dim3(kNT), 0, stream, p);
            else hipLaunchKernelGGL((cache_attention_kernel<dt(), d(), pg(), false, false, false>), grid, dim3(kNT), 0, stream, p);
        });
    }
    if (p.splits > 1) {
        const bool wide = p.splits > kWideSplits;
        int64_t blocks = wide ? rows : (rows + 3) / 4;
        if (blocks > (1 << 20)) blocks = 1 << 20;
        const dim3 merge((unsigned)blocks, (unsigned)kv_heads, (unsigned)batch);
        by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
            if (wide) hipLaunchKernelGGL((cache_attention_merge<dt(), d(), pg(), false, false, 4>), merge, dim3(256), 0, stream, p);
            else hipLaunchKernelGGL((cache_attention_merge<dt(), d(), pg(), false, false, 1>), merge, dim3(256), 0, stream, p);
        });
    }
    return launch_status(what);
}

int64_t h3v_cache_attention_selected_workspace_floats(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t blocks) {
    if (tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || blocks <= 0) return -1;
    return ws_floats(selected_splits(tokens, kv_heads, blocks), tokens, heads, dim);
}

int h3v_cache_attention_selected(int dtype, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                                 const int* selected, int64_t blocks, const int* starts, const int* lens, const int* table,
                                 int64_t batch, int64_t width, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page,
                                 int64_t pages, const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                 const float* v_scale, float scale, uint16_t* out, float* workspace,
                                 int64_t workspace_floats, hipStream_t stream) {
    const char* what = "h3v_cache_attention_selected";
    H3V_REQUIRE(batch > 0 && batch <= 32768 && width > 0 && width <= (1 << 23), "%s: batch or table width out of range", what);
    H3V_REQUIRE(kv_heads > 0, "%s: kv heads must be positive", what);
    AttnParams p = {{starts, lens, table, (int)batch, (int)width, tokens, pages}, q, q_token_stride, q_head_stride, k_cache,
                    v_cache, k_scale, v_scale, scale * 1.4426950408889634f, 1, (int)heads, (int)kv_heads,
                    (int)(heads / kv_heads), out, 1, 1, workspace, selected, (int)blocks, 16, kSplitPages, 0};
    const int rc = check(what, dtype, p, heads, kv_heads, dim, page, scale);
    if (rc) return rc;
    H3V_REQUIRE(selected && aligned(selected, 4), "%s: selected must be a 4-byte aligned array", what);
    H3V_REQUIRE(blocks > 0 && blocks <= 4096, "%s: blocks must be in [1, 4096]", what);
    H3V_REQUIRE(p.group <= 16, "%s: at most 16 query heads per kv head (got %d)", what, p.group);
    const int tile = selected_tile(tokens, batch, width, p.group, blocks);
    if (tile > 1) {
        const int status = launch_selected(what, p, tile, dtype, dim, page, stream);
        return status ? status : launch_status(what);
    }
    p.splits = p.slots = selected_splits(tokens, kv_heads, blocks);
    const int64_t floats = ws_floats(p.splits, tokens, heads, dim);
    H3V_REQUIRE(floats == 0 || (workspace && workspace_floats >= floats && aligned(workspace, 16)),
                "%s: needs a 16-byte aligned workspace of %lld floats", what, (long long)floats);
    H3V_REQUIRE(tokens * kNT <= 0xffffffffll, "%s: too many tokens", what);
    const dim3 grid((unsigned)tokens, (unsigned)kv_heads, (unsigned)p.splits), merge((unsigned)tokens, (unsigned)kv_heads, 1);
    by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
        hipLaunchKernelGGL((cache_attention_kernel<dt(), d(), pg(), true, false, false>), grid, dim3(kNT), 0, stream, p);
        if (p.splits > kWideSplits) hipLaunchKernelGGL((cache_attention_merge<dt(), d(), pg(), true, false, 4>), merge, dim3(256), 0, stream, p);
        else if (p.splits > 1) hipLaunchKernelGGL((cache_attention_merge<dt(), d(), pg(), true, false, 1>), merge, dim3(256), 0, stream, p);
    });
    return launch_status(what);
}

}  // extern "C"
