// Attention over the INT8 K/V cache for long row tiles: prompts and chunks of new tokens (the operator and its other
// kernel: cache_attention.hip).
//
// A workgroup of 8 waves owns 256 * QS query rows ((token, head of the group) pairs) of one kv head, so that one pass over the
// keys serves every head that shares them; wave w the 32 * QS rows from 32 * QS * w.  Keys stream in steps of 64 through
// LDS, three slots of K [64 keys][D] and V^T [D][64 keys] in fp16: every thread loads 16 codes, turns them into fp16 once
// for all waves (the codes are exact there) and stores them.
//
//   S = K . Q^T        v_mfma_f32_32x32x16_f16, A = K rows, B = the wave's Q fragments (registers)
//   softmax            fp32 against a lazy reference maximum; the page's key scale is part of the exponent's factor
//   O^T += V^T . P^T   A = V^T rows, B = P in fp16.  A 16-key group of V^T is stored in the order 0-3, 8-11, 4-7, 12-15, in which
//                      a lane's scores (keys 8 g + 4 (l / 32) + e) already are: P goes from the one product into the
//                      other without leaving its lane.
//
// The page's value scale s_v = f * 2^e, f in [1/2, 1): f joins the weights (exp2(x + log2 f), the row sum takes 1 / f
// back), 2^e the codes, relative to a reference that the accumulators have too: the largest e so far.  fp16 holds codes
// down to 2^-24 of it exactly.  A page further below has a reference of its own, 24 above its e, and the accumulators are brought
// to it before its product and back after it: a power of two each way, exact since fp32 has room for both.
//
// One barrier per step.  On each SIMD a wave of the first half of the workgroup meets one of the second, and their order of
// work is such that the softmax of one runs beside the products of the other: with two sets of 32 rows (QS = 2) the first half
// runs softmax and product of step j and then the scores of step j + 1, the second half the product of step j - 1 and then
// scores and softmax of step j; with one set, where products and softmax differ less, the first half runs scores, softmax and
// product of step j.  (4 x 1797 over 7188, 32 heads of 64: 438 us with this second order, 422 with the first; with one set the first
// order costs 2 to 10%.)  Between barriers j and j + 1 every wave stores its part of the values of step j + 1 and of the keys of step
// j + 1 or, where scores are ahead, j + 2, and loads those after them; the slots they go into were last read before barrier j.
//
// 4 x 1797 over 7188, 32 heads of 64: 404 to 420 us, 800 TFLOP/s, where a library matrix product of as many operations
// takes 252.  The vector units are busy for 58% of the time and the matrix units for 35%; without the staging of codes into
// fp16 it would be 352, without the exponentials 388.  1 x 4096 over 8192, 32 heads of 128: 560 us, 980 TFLOP/s.
#include <algorithm>
#include <type_traits>

#include "cache_attention.hpp"

namespace h3v {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kKB = 64;      // keys of a step
constexpr int kSlots = 3;
constexpr int kNW = 8;       // waves of a workgroup

// 16-byte chunks of a row of `chunks`, placed so that the 32 rows that a fragment read touches cover all banks
template <int CHUNKS>
__device__ __forceinline__ int swz(int row, int chunk) {
    if constexpr (CHUNKS == 8) return chunk ^ ((row >> 1) & 7);
    else return chunk ^ (row & 15);
}

// Barrier of the workgroup's waves where the two halves of them run code of their own.  __syncthreads() may not stand there: it is
// one place that all threads of a workgroup reach together.  s_barrier is an instruction of a wave: it waits until every wave of the workgroup
// has come to one, wherever in the code that is.  Both halves come to 1 + steps of them per tile, and no branch of a wave's
// lanes is around any; the fences are those of __syncthreads().
__device__ __forceinline__ void halves_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
}

// fp16 values of 8 codes times `f` (a power of two from 2^-24 on, or 0), exactly: (1024 + byte) f - 1152 f, with off = -1152 f
__device__ __forceinline__ u32x4 scaled_codes(uint32_t w0, uint32_t w1, f16x2 f, f16x2 off) {
    const uint32_t u0 = w0 ^ 0x80808080u, u1 = w1 ^ 0x80808080u;
    const uint32_t a[4] = {__builtin_amdgcn_perm(0x64646464u, u0, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, u0, 0x04030402u),
                           __builtin_amdgcn_perm(0x64646464u, u1, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, u1, 0x04030402u)};
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, a[i]), f, off));
    return r;
}

// One page's part of a step: its id (-1: not there) and scales.  A value scale of zero (its codes are) or a bad scale (infinite
// or NaN: the scores of the rows that see the page become NaN) stands as a harmless number.
constexpr float kNoScale = 1.0e-37f;
constexpr int kNoExponent = -122;
struct Part {
    int id;
    float ks, vs;
    bool bad;
    int e, f;     // the reference exponent of the codes and of the accumulators, and what the codes have on top of it
};

// Codes are exact down to 2^-24 of the reference.  It drops by at most 75: accumulators stay below 2^(kLazy + kLift) * 127 * 2^30 keys
// < 2^52 of the largest value scale so far, and so below 2^127.  The values of a page below 2^-99 of that scale count as zeros.
constexpr int kExact = 24, kDrop = 75;

// The item-th tile of `rows` rows of the sequences that are long, a sequence's last tiles first; false behind the last.
__device__ __forceinline__ bool long_tile(const AttnParams& p, int rows, int item, int& b, int& tile) {
    const int lane = threadIdx.x & 63;
    for (int at = 0; at < p.s.batch; at += 64) {
        int count = 0;
        if (at + lane < p.s.batch) {
            const Span sp = span_of(p.s, at + lane);
            if (is_long(p, sp)) count = (sp.n * p.group + rows - 1) / rows;
        }
        int upto = count;   // inclusive prefix sum over the lanes
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off, 64);
            if (lane >= off) upto += v;
        }
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (item < all) {
            const int l = __builtin_ctzll(__ballot(upto > item));
            b = at + l;
            tile = __builtin_amdgcn_readlane(upto, l) - 1 - item;
            return true;
        }
        item -= all;
    }
    return false;
}

// MIXED: only the sequences that are long (AttnParams::long_rows), their tiles found by counting.
template <int DT, int D, int P, int QS, bool MIXED>
__global__ __launch_bounds__(64 * kNW) void cache_prefill_kernel(AttnParams p) {
    constexpr int NW = kNW;
    constexpr int NT = 64 * NW, BQ = 32 * QS * NW;
    constexpr int NH = P == 32 ? 2 : 1;                     // pages of a step
    constexpr int KC = D / 16;                              // products of a score tile
    constexpr int DB = D / 32;                              // output tiles
    constexpr int CH = kKB * D / 16;                        // 16-code chunks of K, as many of V
    constexpr int PER = 2 * CH / NT;
    // Fragments read ahead of the products; the compiler by itself reads one and waits for it.  us one at a time / 2 / 4 ahead: 1 x 4096 over 8192, 32 heads
    // of 128 588 / 568 / 566; 4 x 1797 over 7188, 32 heads of 64, 421 / 418 / 464 (registers spill).
    constexpr int kLead = 2;
    constexpr bool AHEAD = QS == 2;                         // scores of a step, and so its keys, a step ahead of its values
    __shared__ __attribute__((aligned(16))) uint16_t kt[kSlots][kKB * D];
    __shared__ __attribute__((aligned(16))) uint16_t vt[kSlots][kKB * D];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5;
    const int sp_i = blockIdx.x;
    const int kvh = blockIdx.y % p.kv_heads;
    int b = blockIdx.z;
    if (b == p.s.batch) {   // rows of no sequence: zeros
        const int64_t lo = p.s.starts[0], hi_row = p.s.starts[p.s.batch], step = (int64_t)gridDim.x * gridDim.y * NT;
        const int64_t row = p.heads * (D / 8);
        for (int64_t e = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * NT + tid; e < p.s.tokens * row; e += step) {
            const int64_t t = e / row;
            if (t < lo || t >= hi_row) *reinterpret_cast<u32x4*>(p.o + 8 * e) = u32x4{0, 0, 0, 0};
        }
        return;
    }
    const int tile_step = gridDim.y / p.kv_heads;
    // the last rows of a causal sequence see the most keys: their tiles first
    for (int item = blockIdx.y / p.kv_heads;; item += tile_step) {
        int tile = 0;
        // sequences whose rows do not overlap have no more tiles than that; starts that decrease end there too
        if constexpr (MIXED)
            if (item > p.s.tokens * p.group / BQ + p.s.batch || !long_tile(p, BQ, item, b, tile)) break;
        const Span span = span_of(p.s, b);
        const int all = span.n * p.group;
        if constexpr (!MIXED) {
            tile = (all + BQ - 1) / BQ - 1 - item;
            if (tile < 0) break;
        }
        const int r0 = tile * BQ, rend = min(all, r0 + BQ);
        const int last = keys_seen(p, span, (rend - 1) / p.group, P);
        const Split sp = split_pages(p, (last + P - 1) / P);
        if (sp_i > 0 && sp_i >= sp.active) continue;
        const int j0 = sp_i * sp.per, j1 = min(sp.pages, j0 + sp.per);
        const int steps = (min(last, j1 * P) - j0 * P + kKB - 1) / kKB;     // <= 0: no key

        const int q0 = r0 + wave * 32 * QS;
        const bool active = q0 < rend;                       // wave-uniform
        int seen[QS], wave_first = 0x7fffffff, wave_last = 0;
        float cq[QS];
        f16x8 qf[QS][KC];
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            const int r = q0 + 32 * qs + (lane & 31), rr = r < rend ? r : rend - 1;
            const int i = rr / p.group, head = kvh * p.group + rr % p.group;
            seen[qs] = keys_seen(p, span, i, P);
            const uint16_t* const src = p.q + (span.row + i) * p.q_ts + head * p.q_hs + 8 * hi;
            u32x4 w[KC];
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) w[kc] = *reinterpret_cast<const u32x4*>(src + 16 * kc);
            cq[qs] = p.c;
            if constexpr (DT == kF16) {
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) qf[qs][kc] = __builtin_bit_cast(f16x8, w[kc]);
            } else {
                float top = 0.0f;
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    float v[8];
                    unpack8<DT>(w[kc], v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(v[e]));
                }
                top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
                const int ex = __builtin_amdgcn_frexp_expf(top);
                cq[qs] = __builtin_amdgcn_ldexpf(p.c, ex);
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    float v[8];
                    unpack8<DT>(w[kc], v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = __builtin_amdgcn_ldexpf(v[e], -ex);
                    qf[qs][kc] = __builtin_bit_cast(f16x8, pack8<kF16>(v));
                }
            }
        }
        if (active) {
            wave_first = keys_seen(p, span, q0 / p.group, P);
            wave_last = keys_seen(p, span, (min(rend, q0 + 32 * QS) - 1) / p.group, P);
        }

        // pages of the split, 64 at a time: ids and scales one page per lane
        int pg_base = -64, pg_id = -1, pg_e = 0;              // pg_e: exponent of the value scale, kBadPage more where a scale is bad
        float pg_ks = 0.0f, pg_vs = 0.0f;
        constexpr int kBadPage = 4096;
        int eref = -126;                                      // largest value exponent of the steps so far
        auto part_of = [&](int j) {                           // page j0 + j
            if (j - pg_base >= 64) {
                pg_base = j;
                const int mine = j0 + j + lane;
                pg_id = mine < j1 ? page_id(p.s, b, mine) : -1;
                pg_ks = pg_vs = 0.0f;
                if (pg_id >= 0) {
                    pg_ks = p.ks[(int64_t)pg_id * p.kv_heads + kvh];
                    pg_vs = p.vs[(int64_t)pg_id * p.kv_heads + kvh];
                }
                const bool bad = !(pg_ks - pg_ks == 0.0f && pg_vs - pg_vs == 0.0f);
                pg_ks = pg_ks - pg_ks == 0.0f ? pg_ks : 1.0f;
                pg_vs = pg_vs - pg_vs == 0.0f ? __builtin_fmaxf(pg_vs, kNoScale) : kNoScale;
                pg_e = __builtin_amdgcn_frexp_expf(pg_vs) + (bad ? kBadPage : 0);
            }
            const int n = j - pg_base;
            Part r;
            r.id = __builtin_amdgcn_readlane(pg_id, n);
            r.ks = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pg_ks), n));
            r.vs = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pg_vs), n));
            const int e = __builtin_amdgcn_readlane(pg_e, n);
            r.bad = e > kBadPage / 2;
            const int own = r.bad ? e - kBadPage : e;
            eref = max(eref, own);
            r.e = own >= eref - kExact || own == kNoExponent ? eref : max(own + kExact, eref - kDrop);
            r.f = own - r.e;
            return r;
        };
        struct Step {
            Part h[NH];
        };
        auto sound = [](const Step& s) {                      // pages that are there, with finite scales
            return s.h[0].id >= 0 && !s.h[0].bad && s.h[NH - 1].id >= 0 && !s.h[NH - 1].bad;
        };
        auto step_of = [&](int j) {
            Step s;
            s.h[0] = part_of(NH == 2 ? 2 * j : (P == 128 ? j >> 1 : j));
            if constexpr (NH == 2) s.h[1] = part_of(2 * j + 1);
            return s;
        };

        // this thread's chunks: K: key, 16 dims; V: dim, 16 keys
        struct Chunks {
            u32x4 w[PER];
        };
        auto load = [&](Chunks& reg, bool keys, const Step& sk, int jk, bool values, const Step& sv, int jv) {
            const int koff = P == 128 ? (jk & 1) * kKB : 0, voff = P == 128 ? (jv & 1) * kKB : 0;
            const int k0 = sk.h[0].id, k1 = sk.h[NH - 1].id, v0 = sv.h[0].id, v1 = sv.h[NH - 1].id;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = tid + i * NT;
                if (c < CH) {
                    if (!keys) continue;
                    const int key = c / (D / 16), dch = c % (D / 16);
                    const int h = NH == 2 ? key >> 5 : 0, id = NH == 2 && h ? k1 : k0;
                    const int64_t ph = (int64_t)(id < 0 ? 0 : id) * p.kv_heads + kvh;
                    reg.w[i] = *reinterpret_cast<const u32x4*>(p.k + ph * (P * D) + (koff + (NH == 2 ? key & 31 : key)) * D + 16 * dch);
                } else {
                    if (!values) continue;
                    const int d = (c - CH) >> 2, kch = (c - CH) & 3;
                    const int h = NH == 2 ? kch >> 1 : 0, id = NH == 2 && h ? v1 : v0;
                    const int64_t ph = (int64_t)(id < 0 ? 0 : id) * p.kv_heads + kvh;
                    reg.w[i] = *reinterpret_cast<const u32x4*>(p.v + ph * (P * D) + d * P + voff + 16 * (NH == 2 ? kch & 1 : kch));
                }
            }
        };
        auto store = [&](const Chunks& reg, bool keys, int kslot, bool values, const Step& sv, int vslot) {
            const int f0 = sv.h[0].f, f1 = sv.h[NH - 1].f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = tid + i * NT;
                if (c < CH) {
                    if (!keys) continue;
                    const int key = c / (D / 16), dch = c % (D / 16);
                    const f16x8 lo = codes_to_f16x8(reg.w[i][0], reg.w[i][1]), up = codes_to_f16x8(reg.w[i][2], reg.w[i][3]);
                    uint16_t* const row = kt[kslot] + key * D;
                    *reinterpret_cast<f16x8*>(row + 8 * swz<D / 8>(key, 2 * dch)) = lo;
                    *reinterpret_cast<f16x8*>(row + 8 * swz<D / 8>(key, 2 * dch + 1)) = up;
                } else {
                    if (!values) continue;
                    const int d = (c - CH) >> 2, kch = (c - CH) & 3;
                    // rounded first: below 2^-24 the factor and the offset are zeros together
                    const f16 fh = (f16)__builtin_amdgcn_ldexpf(1.0f, NH == 2 && (kch >> 1) ? f1 : f0), oh = (f16)-1152.0f * fh;
                    const f16x2 f2 = {fh, fh}, off = {oh, oh};
                    uint16_t* const row = vt[vslot] + d * kKB;
                    *reinterpret_cast<u32x4*>(row + 8 * swz<8>(d, 2 * kch)) = scaled_codes(reg.w[i][0], reg.w[i][2], f2, off);
                    *reinterpret_cast<u32x4*>(row + 8 * swz<8>(d, 2 * kch + 1)) = scaled_codes(reg.w[i][1], reg.w[i][3], f2, off);
                }
            }
        };

        auto work = [&](auto first) {
        constexpr bool FIRST = first();
        f32x16 o[QS][DB];
        float m[QS], l[QS];
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
#pragma unroll
            for (int d = 0; d < DB; ++d) o[qs][d] = f32x16{};
            m[qs] = -kInf;
            l[qs] = 0.0f;
        }
        bool far = false;                                    // some row's reference is past kFar (the same for all lanes)
        uint32_t pk[QS][2][8];

        f32x16 x[QS][2];
        auto scores = [&](int slot) {
            const uint16_t* const kb = kt[slot];
            auto fragment = [&](int n) {                     // keys 32 (n / KC) .., dims 16 (n % KC) ..
                const int row = 32 * (n / KC) + (lane & 31);
                return *reinterpret_cast<const f16x8*>(kb + row * D + 8 * swz<D / 8>(row, 2 * (n % KC) + hi));
            };
            f16x8 a[kLead + 1];
#pragma unroll
            for (int n = 0; n < kLead; ++n) a[n] = fragment(n);
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) x[qs][0] = x[qs][1] = f32x16{};
#pragma unroll
            for (int n = 0; n < 2 * KC; ++n) {
                if (n + kLead < 2 * KC) a[(n + kLead) % (kLead + 1)] = fragment(n + kLead);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs)
                    x[qs][n / KC] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n % (kLead + 1)], qf[qs][n % KC], x[qs][n / KC], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // weights of step j's scores
        auto weigh = [&](const Step& s, int j) {
            const int key0 = j0 * P + j * kKB;
            if (!(key0 + kKB <= wave_first && sound(s))) {
#pragma unroll
                for (int kh = 0; kh < 2; ++kh) {
                    const Part& h = s.h[NH == 2 ? kh : 0];
                    const float poison = h.bad ? __builtin_nanf("") : 0.0f;
#pragma unroll
                    for (int qs = 0; qs < QS; ++qs) {
                        const int lim = (h.id >= 0 ? seen[qs] : 0) - key0 - 32 * kh - 4 * hi;
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[qs][kh][r] = 8 * (r >> 2) + (r & 3) < lim ? x[qs][kh][r] + poison : -kInf;
                    }
                }
            }
            // a factor that is too small for fp32 keeps a masked score at minus infinity
            float kf[QS][NH], lm[NH], im[NH];
#pragma unroll
            for (int h = 0; h < NH; ++h) {
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) kf[qs][h] = __builtin_fmaxf(s.h[h].ks * cq[qs], 1.0e-37f);
                const float f = __builtin_amdgcn_frexp_mantf(s.h[h].vs);
                lm[h] = __builtin_amdgcn_logf(f);
                im[h] = 1.0f / f;
            }
            bool up = false;
            float top[QS];
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
                float t[2];
#pragma unroll
                for (int kh = 0; kh < 2; ++kh) {
                    t[kh] = x[qs][kh][0];
#pragma unroll
                    for (int r = 1; r < 16; ++r) t[kh] = __builtin_fmaxf(t[kh], x[qs][kh][r]);
                }
                top[qs] = NH == 2 ? __builtin_fmaxf(t[0] * kf[qs][0], t[1] * kf[qs][NH - 1]) : __builtin_fmaxf(t[0], t[1]) * kf[qs][0];
                up |= top[qs] > m[qs] + kLazy;
            }
            if (__ballot(up)) {
                bool past = false;
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) {
                    const float m_new = __builtin_fmaxf(m[qs], __builtin_fmaxf(top[qs], __shfl_xor(top[qs], 32, 64)));
                    const float alpha = m[qs] == m_new ? 1.0f : __builtin_amdgcn_exp2f(m[qs] - m_new);
                    m[qs] = m_new;
                    l[qs] *= alpha;
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[qs][d] *= alpha;
                    past |= is_far(m[qs]);
                }
                far = __ballot(past) != 0;
            }
            if (far) {                                       // weights from rounded scores less the reference
#pragma unroll
                for (int qs = 0; qs < QS; ++qs)
#pragma unroll
                    for (int kh = 0; kh < 2; ++kh) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[qs][kh][r] = x[qs][kh][r] * kf[qs][NH == 2 ? kh : 0] - (m[qs] == -kInf ? 0.0f : m[qs]);
                    }
#pragma unroll
                for (int qs = 0; qs < QS; ++qs)
#pragma unroll
                    for (int h = 0; h < NH; ++h) kf[qs][h] = 1.0f;
            }
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
                const float base = (far || m[qs] == -kInf ? 0.0f : m[qs]) - kLift;
                float sum = 0.0f;
#pragma unroll
                for (int kh = 0; kh < 2; ++kh) {
                    const int h = NH == 2 ? kh : 0;
                    const float off = lm[h] - base;
                    if (NH == 2) sum = 0.0f;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[qs][kh][4 * g + e], kf[qs][h], off));
                        pk[qs][kh][2 * g] = pack2<kF16>(w[0], w[1]);
                        pk[qs][kh][2 * g + 1] = pack2<kF16>(w[2], w[3]);
                        const f16x2 one = {(f16)1.0f, (f16)1.0f};
                        sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk[qs][kh][2 * g]), one, sum, false);
                        sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk[qs][kh][2 * g + 1]), one, sum, false);
                    }
                    if (NH == 2 || kh == 1) l[qs] = __builtin_fmaf(sum, im[h], l[qs]);
                }
            }
        };
        // O^T += V^T . P^T
        int oe = -126;                                       // the reference exponent of o
        auto product = [&](int e0, int e1, int slot) {       // of the step's first and last page
            const uint16_t* const vb = vt[slot];
            auto fragment = [&](int n) {                     // dims 32 (n % DB) .., keys 16 (n / DB) ..
                const int row = 32 * (n % DB) + (lane & 31);
                return *reinterpret_cast<const f16x8*>(vb + row * kKB + 8 * swz<8>(row, 2 * (n / DB) + hi));
            };
            f16x8 a[kLead + 1];
#pragma unroll
            for (int n = 0; n < kLead; ++n) a[n] = fragment(n);
#pragma unroll
            for (int n = 0; n < 4 * DB; ++n) {
                const int c = n / DB;
                // per page: a row that sees the first one alone has its values to their own exponent
                const int e = c < 2 ? e0 : e1;
                if ((n == 0 || (NH == 2 && n == 2 * DB)) && e != oe) {
                    const float drop = __builtin_amdgcn_ldexpf(1.0f, oe - e);
#pragma unroll
                    for (int qs = 0; qs < QS; ++qs)
#pragma unroll
                        for (int d = 0; d < DB; ++d) o[qs][d] *= drop;
                    oe = e;
                }
                if (n + kLead < 4 * DB) a[(n + kLead) % (kLead + 1)] = fragment(n + kLead);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) {
                    const int g = 4 * (c & 1);
                    const u32x4 w = {pk[qs][c >> 1][g], pk[qs][c >> 1][g + 1], pk[qs][c >> 1][g + 2], pk[qs][c >> 1][g + 3]};
                    o[qs][n % DB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[n % (kLead + 1)], __builtin_bit_cast(f16x8, w), o[qs][n % DB], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };

        if (steps > 0) {
            // step j and those after it; steps behind the last have no pages
            Step cur = step_of(0), s1 = step_of(1), s2 = s1, s3 = s1;
            Chunks next;
            {
                Chunks now;
                load(now, true, cur, 0, true, cur, 0);
                if constexpr (AHEAD) {
                    s2 = step_of(2);
                    load(next, steps > 1, s1, 1, false, s1, 1);
                }
                store(now, true, 0, true, cur, 0);
                if constexpr (AHEAD) store(next, steps > 1, 1, false, s1, 1);
            }
            load(next, steps > 1 + AHEAD, AHEAD ? s2 : s1, 1 + AHEAD, steps > 1, s1, 1);
            int slot = 0, up1 = 1, up2 = 2;                   // slots of j, j + 1, j + 2
            int pe0 = -126, pe1 = -126;
            auto sees = [&](int u) { return j0 * P + u * kKB < wave_last; };
            halves_barrier();
            if (FIRST && AHEAD && sees(0)) scores(0);
            for (int j = 0; j < steps; ++j) {
                store(next, j + 1 + AHEAD < steps, AHEAD ? up2 : up1, j + 1 < steps, s1, up1);
                if constexpr (AHEAD) s3 = step_of(j + 3);
                else s2 = step_of(j + 2);
                load(next, j + 2 + AHEAD < steps, AHEAD ? s3 : s2, j + 2 + AHEAD, j + 2 < steps, s2, j + 2);
                if constexpr (FIRST) {
                    if (sees(j)) {
                        if constexpr (!AHEAD) scores(slot);
                        weigh(cur, j);
                        product(cur.h[0].e, cur.h[NH - 1].e, slot);
                    }
                    if (AHEAD && j + 1 < steps && sees(j + 1)) scores(up1);
                } else {
                    if (j > 0 && sees(j - 1)) product(pe0, pe1, up2);
                    if (sees(j)) {
                        scores(slot);
                        weigh(cur, j);
                    }
                    pe0 = cur.h[0].e;
                    pe1 = cur.h[NH - 1].e;
                }
                cur = s1;
                s1 = s2;
                if constexpr (AHEAD) s2 = s3;
                const int t = slot;
                slot = up1;
                up1 = up2;
                up2 = t;
                halves_barrier();
            }
            if (!FIRST && sees(steps - 1)) product(pe0, pe1, up2);
        }

        // lane l holds row q0 + 32 qs + l % 32, dims 32 d + 8 g + 4 hi + e
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            const int r = q0 + 32 * qs + (lane & 31);
            const float lt = l[qs] + __shfl_xor(l[qs], 32, 64);
            if (r >= rend) continue;
            const int64_t row = (span.row + r / p.group) * p.heads + kvh * p.group + r % p.group;
            if (sp.active > 1) {
                const int64_t at = (int64_t)sp_i * p.s.tokens * p.heads + row;
                float* const dst = p.part + at * D + 4 * hi;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(o[qs][d][4 * g + e], oe - kOutDrop);
                        *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * g) = v;
                    }
                if (hi == 0) {
                    float* const pml = p.part + (int64_t)p.slots * p.s.tokens * p.heads * D + 2 * at;
                    pml[0] = m[qs];
                    pml[1] = lt;
                }
                continue;
            }
            const float inv = m[qs] == -kInf && lt == 0.0f ? 0.0f : 1.0f / lt;
            uint16_t* const dst = p.o + row * D + 4 * hi;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(o[qs][d][4 * g + e] * inv, oe);
                    *reinterpret_cast<uint2*>(dst + 32 * d + 8 * g) = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
                }
        }
        };
        // each half of the waves to the tile's end by itself: registers of the two need not agree anywhere.  `wave` and `steps` are
        // the same for all lanes of a wave, `steps` for all waves (halves_barrier)
        if (wave < NW / 2) work(std::true_type{});
        else work(std::false_type{});
        __syncthreads();   // the next tile's first store waits for this tile's last reads
    }
}

template <int DT, int D, int P, bool MIXED>
void launch_shape(const AttnParams& p, dim3 grid, hipStream_t stream) {
    if constexpr (D == 64)
        if (p.tile_rows == 512) {
            hipLaunchKernelGGL((cache_prefill_kernel<DT, D, P, 2, MIXED>), grid, dim3(64 * kNW), 0, stream, p);
            return;
        }
    hipLaunchKernelGGL((cache_prefill_kernel<DT, D, P, 1, MIXED>), grid, dim3(64 * kNW), 0, stream, p);
}

}  // namespace

// At dim 64 two sets of 32 rows per wave read each key and value fragment once for both.  A CU holds one workgroup of either
// form (by the registers of its 8 waves), so there have to be twice the rows: the larger one pays where it makes two rounds on the
// 256 CUs, or fills one without causal rows, whose longest tile would be the round (us, 512 / 256 rows; batch x new over length, 32 heads):
//   4 x 1797 over 7188: 413 / 513, causal 373 / 445;  1 x 4096: 160 / 194, causal 148 / 110;  3 x 1100: 85 / 64, causal 57 / 53
//
// The keys are split where that shortens the rounds by more than the splits' outputs cost, written and joined (4 TB/s and a
// launch of 5 us): s splits take ceil(s units / 256) rounds of 1 / s of the steps each.  us, one split / by this estimate, 8 kv
// heads of 128, four heads each: 1 x 1300 over 8000 243 / 203, 4 x 300 over 4000 126 / 105, 10 x 100 over 3000 96 / 87.  A table may be much wider than its sequences are long: a split has at least the
// steps that pay for its outputs three times over, and shorter sequences are not split.
PrefillPlan plan_prefill(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t rows, int64_t width, int64_t page,
                         int64_t dim, bool causal, bool mixed) {
    constexpr int64_t kCUs = 256;
    // of sequences that differ, one's rows, with a token left for each of the others
    const int64_t most = std::max(rows / batch, (tokens - std::min(tokens, batch - 1)) * (heads / kv_heads));
    auto units = [&](int64_t t) { return kv_heads * (mixed ? (most + t - 1) / t : batch * ((rows + t - 1) / t)); };
    PrefillPlan r = {256, 1, 4};
    const int64_t u512 = units(512);
    if (dim == 64 && (u512 >= 2 * kCUs || (!causal && u512 <= kCUs && 8 * u512 >= 7 * kCUs))) r.tile_rows = 512;
    const int64_t u = units(r.tile_rows);
    const double steps = (double)width * page / kKB, step_us = r.tile_rows == 512 ? 1.9 : (dim == 64 ? 1.15 : 2.1);
    const double join_us = (double)tokens * heads * dim * 8 / 4e6;      // of one split's outputs
    double best = 0.0;
    for (int s = 1; s <= 16 && (s == 1 || s * r.least <= width); ++s) {
        const double us = (double)((u * s + kCUs - 1) / kCUs) * (steps / s) * step_us + (s > 1 ? 5.0 + s * join_us : 0.0);
        if (s == 1 || us < best) {
            best = us;
            r.splits = s;
        }
    }
    const int64_t least = (int64_t)(3.0 * join_us / step_us * kKB / page);
    if (least > r.least) r.least = (int)(least < width ? least : width);
    return r;
}

void launch_prefill(const AttnParams& p, int dtype, int64_t dim, int64_t page, int64_t rows, hipStream_t stream) {
    int64_t tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    if (tiles > 65535 / p.kv_heads) tiles = 65535 / p.kv_heads;
    // of several sequences, the 16-row tiles' launch clears the rows of none
    const dim3 grid((unsigned)p.splits, (unsigned)(tiles * p.kv_heads), p.long_rows > 0 ? 1u : (unsigned)(p.s.batch + 1));
    by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
        if (p.long_rows > 0) launch_shape<dt(), d(), pg(), true>(p, grid, stream);
        else launch_shape<dt(), d(), pg(), false>(p, grid, stream);
    });
}

}  // namespace h3v
