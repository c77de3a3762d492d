// Sixteen query rows of one kv head against pages of the INT8 K/V cache, by one wave, all in registers (the mathematics:
// cache_attention.hip).
#pragma once

#include "cache_attention.hpp"

namespace h3v {

// Loads of codes; STREAM: marked non-temporal, for pages that one workgroup reads.
template <bool STREAM, typename T>
__device__ __forceinline__ T load_codes(const int8_t* at) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T*>(at));
    else return *reinterpret_cast<const T*>(at);
}

template <int DT, int D, int P>
struct RowTile {
    static constexpr int KT = P < 64 ? 32 : 64;    // keys of a step
    static constexpr int NT = KT / 16;             // score tiles of a step
    static constexpr int NL = D / 64;              // 16-byte loads of a key per lane
    static constexpr int ND = D / 16;              // output tiles
    static constexpr int NSUB = P / KT;            // steps of a page
    static constexpr int VW = KT / 16;             // words of a lane's value codes

    struct Codes {
        u32x4 k[NT][NL];
        uint32_t v[ND][VW];
    };

    int col, g;            // row of this lane, and its quarter of a step's keys
    f16x8 qf[2 * NL];      // slot (L, step s, group g, e) is dim 64 L + 16 g + 8 s + e
    float c;               // scale * log2(e), times the power of two that bf16 queries were divided by
    f32x4 o[ND];
    float add, l;          // the exponents' addend: kLift minus the reference maximum (infinite without one); the row's sum
    bool any;              // this lane's row saw a key
    bool far;              // some row's reference is past kFar (the same for all lanes)

    // row: the query row of this lane's column.  Only loads; set_rows() makes fragments of them.
    __device__ __forceinline__ void load_rows(const uint16_t* row) {
        const int lane = threadIdx.x & 63;
        col = lane & 15;
        g = lane >> 4;
#pragma unroll
        for (int f = 0; f < 2 * NL; ++f) qf[f] = *reinterpret_cast<const f16x8*>(row + 16 * g + 64 * (f >> 1) + 8 * (f & 1));
    }

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        add = kInf;
        l = 0.0f;
        any = false;
        far = false;
    }

    __device__ __forceinline__ void set_rows(float scale) {
        c = scale;
        if constexpr (DT == kBF16) {
            float v[2 * NL][8], top = 0.0f;
#pragma unroll
            for (int f = 0; f < 2 * NL; ++f) {
                unpack8<DT>(__builtin_bit_cast(u32x4, qf[f]), v[f]);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, __builtin_fabsf(v[f][e]));
            }
            top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
            const int ex = __builtin_amdgcn_frexp_expf(top);
            c = __builtin_amdgcn_ldexpf(c, ex);
#pragma unroll
            for (int f = 0; f < 2 * NL; ++f) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[f][e] = __builtin_amdgcn_ldexpf(v[f][e], -ex);
                qf[f] = __builtin_bit_cast(f16x8, pack8<kF16>(v[f]));
            }
        }
    }

    // codes of step `sub` of the (page, head) pair ph
    template <bool STREAM>
    __device__ __forceinline__ void load(Codes& w, const int8_t* k, const int8_t* v, int64_t ph, int sub) const {
        const int8_t* const kp = k + ph * (P * D) + (sub * KT + KT / 4 * (col >> 2) + (col & 3)) * D + 16 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int L = 0; L < NL; ++L) w.k[t][L] = load_codes<STREAM, u32x4>(kp + 4 * t * D + 64 * L);
        const int8_t* const vp = v + ph * (P * D) + col * P + sub * KT + KT / 4 * g;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            if constexpr (VW == 4) {
                const u32x4 x = load_codes<STREAM, u32x4>(vp + d * 16 * P);
#pragma unroll
                for (int e = 0; e < 4; ++e) w.v[d][e] = x[e];
            } else {
                const u32x2 x = load_codes<STREAM, u32x2>(vp + d * 16 * P);
                w.v[d][0] = x[0];
                w.v[d][1] = x[1];
            }
        }
    }

    // the step of the keys key0 .., of which this lane's row sees those below `seen`; vs: the page's value scale times 2^-kOutDrop
    __device__ __forceinline__ void attend(const Codes& w, int key0, float ks, float vs, int seen) {
        // a factor that is too small for fp32 keeps a masked score at minus infinity
        const float kc = ks * c < 1.0e-37f ? 1.0e-37f : ks * c;
        f32x4 x[NT];
        float top = -kInf;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            x[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int L = 0; L < NL; ++L)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16x8(w.k[t][L][2 * s], w.k[t][L][2 * s + 1]), qf[2 * L + s],
                                                                  x[t], 0, 0, 0);
        }
        // rows that see all of the step or none of it need no look at its single keys
        if (__ballot(key0 < seen && key0 + KT > seen)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + KT / 4 * g + 4 * t + e >= seen) x[t][e] = -kInf;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = __builtin_fmaxf(top, x[t][e]);
        const bool sees = key0 < seen;
        any |= sees;
        top = sees ? top * kc : -kInf;
        if (__ballot(top + add > kLazy + kLift)) {
            top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
            const float lower = __builtin_fminf(add, kLift - top);
            const float alpha = add == lower ? 1.0f : __builtin_amdgcn_exp2f(lower - add);
            add = lower;
            far = __ballot(is_far(add)) != 0;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[d] *= alpha;
        }
        // a row that sees no key of the step takes nothing from it, not even from a scale that is NaN
        float factor = sees ? kc : 1.0f;
        const float from = sees ? add : -kInf, vrow = sees ? vs : 0.0f;
        if (far) {
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] *= factor;
            factor = 1.0f;
        }
        uint32_t pk[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) e4[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][e], factor, from));
            pk[t][0] = pack2<kF16>(e4[0], e4[1]);
            pk[t][1] = pack2<kF16>(e4[2], e4[3]);
            const f16x2 one = {(f16)1.0f, (f16)1.0f};
            l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk[t][0]), one, l, false);
            l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pk[t][1]), one, l, false);
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < NT / 2; ++s) {
                const u32x4 bw = {pk[2 * s][0], pk[2 * s][1], pk[2 * s + 1][0], pk[2 * s + 1][1]};
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_f16x8(w.v[d][2 * s], w.v[d][2 * s + 1]),
                                                             __builtin_bit_cast(f16x8, bw), acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] = __builtin_fmaf(acc[e], vrow, o[d][e]);
        }
    }

    // Runs `steps` steps, `load_step(w)` and `attend_step(w)` in the steps' order, over two sets of registers in turn: the
    // next step's loads are ahead of this step's work.  No load sits behind a branch within the loop: the wait counts of
    // the path without it would hold for the other one too.
    template <typename W, typename L, typename A>
    __device__ __forceinline__ static void run(int steps, L&& load_step, A&& attend_step) {
        if (steps <= 0) return;
        W w0, w1;
        load_step(w0);
        int u = 0;
        for (; u + 2 < steps; u += 2) {
            load_step(w1);
            __builtin_amdgcn_sched_barrier(0);
            attend_step(w0);
            load_step(w0);
            __builtin_amdgcn_sched_barrier(0);
            attend_step(w1);
        }
        if (u + 1 < steps) {
            load_step(w1);
            __builtin_amdgcn_sched_barrier(0);
            attend_step(w0);
            attend_step(w1);
        } else {
            attend_step(w0);
        }
    }
};

// The parts of a workgroup's NW waves for 16 rows, joined through LDS.
template <int D, int NW>
struct Joined {
    float o[NW][16][D + 4];
    float ml[NW][16][2];

    template <typename TILE>
    __device__ __forceinline__ void put(const TILE& t, int wave) {
        // a row that saw no key takes nothing from a query that is infinite or NaN either
        float l = t.any ? t.l : 0.0f;
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(&o[wave][t.col][16 * d + 4 * t.g]) = t.any ? t.o[d] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (t.g == 0) {
            ml[wave][t.col][0] = -t.add;     // the maximum less kLift, as in every part
            ml[wave][t.col][1] = l;
        }
    }

    // dims d .. d + 3 of row r: unnormalised output, reference maximum, sum
    __device__ __forceinline__ f32x4 get(int r, int d, float& top, float& sum) const {
        top = -kInf;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = __builtin_fmaxf(top, ml[w][r][0]);
        f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = part_weight(ml[w][r][0], top);
            sum = __builtin_fmaf(f, ml[w][r][1], sum);
            const f32x4 v = *reinterpret_cast<const f32x4*>(&o[w][r][d]);
#pragma unroll
            for (int x = 0; x < 4; ++x) out[x] = __builtin_fmaf(f, v[x], out[x]);
        }
        return out;
    }
};

// What brings a row's unnormalised output to its value: 2^kOutDrop over the row's sum; a row that saw no key gets 0.
__device__ __forceinline__ float row_inverse(float top, float sum) {
    return top == -kInf && sum == 0.0f ? 0.0f : (float)(1 << kOutDrop) / sum;
}

template <int DT>
__device__ __forceinline__ void put_row(uint16_t* at, const f32x4& v, float inv) {
    *reinterpret_cast<u32x2*>(at) = u32x2{pack2<DT>(v[0] * inv, v[1] * inv), pack2<DT>(v[2] * inv, v[3] * inv)};
}

}  // namespace h3v
