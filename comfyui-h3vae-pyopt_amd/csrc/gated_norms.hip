// The norm behind a block, the block's gate and residual scale, and the norm before the next block, in one pass:
//
//   z = y * rsqrt(mean(y^2) + eps) * w_post        (no w_post: z = y)
//   h = x + alpha * gate * z                       (no gate: 1)
//   n = h * rsqrt(mean(h^2) + eps) * w_pre         from the unrounded fp32 h
//
// h, n in the inputs' type, or n as int8 rows: s = max(amax / 127, 1e-30), q = rint(n * fl(1 / s)), what the INT8
// linears take.  Everything between the loads and the one rounding of each output is fp32.
//
// A row lives in registers from its one read to its one write: W waves per row (1, or all 4 of a workgroup), lane
// l of wave p holding the 8 values at ((c * W + p) * 64 + l) * 8 of each chunk c, 16-byte loads and stores.
//
// Bound by memory: 7188 x 2048 fp16, 118 MB, in 23.1 us; 16383 x 2560 bf16 with a gate per row, 419 MB, in 77 us.
#include <type_traits>

#include "h3v_half.hpp"
#include "h3v_abi.hpp"

namespace h3v {
namespace {

constexpr int kNT = 256;

struct NormParams {
    const uint16_t *x, *y, *gate, *post, *pre;
    float alpha, eps;
    int64_t m, rows_per_gate;
    int k;
    uint16_t *h, *n;
    int8_t* q;
    float* scale;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Sum over a row of the lanes' sums.  One wave: a sum for each of up to two chunks, joined as two waves would join theirs, so that a
// row's bits do not depend on how many waves it has.
template <int W, int N>
__device__ __forceinline__ float row_sum(const float (&v)[N], float* red, int wave) {
    static_assert(W == 1 ? N <= 2 : N == 1);
    const float s = wave_sum(v[0]);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) red[wave] = s;
        __syncthreads();
        return (red[0] + red[1]) + (red[2] + red[3]);
    }
    if constexpr (N > 1) return s + wave_sum(v[N - 1]);
    return s;
}

// How a call uses the caches, by the bytes of its outputs (gated norms alone / with a sum and a matrix product that read h and n,
// us, plain against streamed stores):
//   up to 32 MB, the L2s together: stores streamed, so that none are left to write back at the kernel's end
//     (1000 x 2048: 7.4 / 5.8, with its readers 30.2 / 29.6; 2000 x 2048: 37.8 / 36.5 with them)
//   up to 256 MB, the Infinity Cache: plain; the next kernels find them there (16383 x 2560: 79 / 75 alone, but 312 / 318
//     with its readers)
//   beyond: loads and stores streamed (32768 x 4096: 1138 / 1117 with its readers)
enum class Use { Stores, Plain, Both };
constexpr int64_t kL2Bytes = 32 << 20, kCacheBytes = 256 << 20;

template <bool STREAM>
__device__ __forceinline__ u32x4 read16(const uint16_t* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    else return *reinterpret_cast<const u32x4*>(p);
}
template <bool STREAM, typename T>
__device__ __forceinline__ void write_out(void* p, const T& v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<T*>(p));
    else *reinterpret_cast<T*>(p) = v;
}

template <int DT, int W, int NCH, bool POST, bool Q8, Use USE>
__global__ __launch_bounds__(kNT) void gated_norms_kernel(NormParams p) {
    __shared__ float red[3][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
    if (row >= p.m) return;   // W = 4: the whole workgroup
    const int part = W == 1 ? 0 : wave;
    const int64_t base = row * p.k;
    const uint16_t* const gate = p.gate ? p.gate + row / p.rows_per_gate * p.k : nullptr;
    const float inv_k = 1.0f / (float)p.k;

    u32x4 xw[NCH], yw[NCH], gw[NCH];
    int col[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        col[c] = ((c * W + part) * 64 + lane) * 8;
        if (col[c] < p.k) {
            xw[c] = read16<USE == Use::Both>(p.x + base + col[c]);
            yw[c] = read16<USE == Use::Both>(p.y + base + col[c]);
            if (gate) gw[c] = *reinterpret_cast<const u32x4*>(gate + col[c]);
        } else {
            xw[c] = yw[c] = gw[c] = u32x4{0, 0, 0, 0};
        }
    }
    constexpr int NS = W == 1 ? NCH : 1;                 // sums of a lane
    float f = p.alpha;
    if constexpr (POST) {
        float ss[NS] = {};
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float v[8];
            unpack8<DT>(yw[c], v);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[c % NS] = __builtin_fmaf(v[e], v[e], ss[c % NS]);
        }
        f *= rsqrt_rn(row_sum<W>(ss, red[0], wave) * inv_k + p.eps);
    }
    float h[NCH][8];
    float ss[NS] = {};
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        float xv[8], yv[8], gv[8], wv[8];
        unpack8<DT>(xw[c], xv);
        unpack8<DT>(yw[c], yv);
        if (gate) unpack8<DT>(gw[c], gv);
        if (POST && col[c] < p.k) unpack8<DT>(*reinterpret_cast<const u32x4*>(p.post + col[c]), wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float z = yv[e] * f;
            if (POST) z *= col[c] < p.k ? wv[e] : 0.0f;
            h[c][e] = gate ? __builtin_fmaf(z, gv[e], xv[e]) : xv[e] + z;
            ss[c % NS] = __builtin_fmaf(h[c][e], h[c][e], ss[c % NS]);
        }
        if (col[c] < p.k) write_out<USE != Use::Plain>(p.h + base + col[c], pack8<DT>(h[c]));
    }
    const float inv = rsqrt_rn(row_sum<W>(ss, red[1], wave) * inv_k + p.eps);
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        float wv[8] = {};
        if (col[c] < p.k) unpack8<DT>(*reinterpret_cast<const u32x4*>(p.pre + col[c]), wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[c][e] = (h[c][e] * inv) * wv[e];
            if (Q8) {
                amax = __builtin_fmaxf(amax, __builtin_fabsf(h[c][e]));
                bad |= h[c][e] != h[c][e];
            }
        }
        if (!Q8 && col[c] < p.k) write_out<USE != Use::Plain>(p.n + base + col[c], pack8<DT>(h[c]));
    }
    if constexpr (Q8) {
        amax = wave_max(amax);
        if (__ballot(bad)) amax = __builtin_nanf("");
        if constexpr (W > 1) {
            if (lane == 0) red[2][wave] = amax;
            __syncthreads();
            float all = 0.0f;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all = __builtin_fmaxf(all, red[2][i]);
                nan |= red[2][i] != red[2][i];
            }
            amax = nan ? __builtin_nanf("") : all;
        }
        const float s = code_scale(amax), r = 1.0f / s;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (col[c] >= p.k) continue;
            write_out<USE != Use::Plain>(p.q + base + col[c], u32x2{codes4(h[c][0] * r, h[c][1] * r, h[c][2] * r, h[c][3] * r),
                                                                    codes4(h[c][4] * r, h[c][5] * r, h[c][6] * r, h[c][7] * r)});
        }
        if (part == 0 && lane == 0) p.scale[row] = s;
    }
}

template <int DT, int W, int NCH, Use USE>
void launch_use(const NormParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)((p.m + 4 / W - 1) / (4 / W))), block(kNT);
    if (p.post && p.q) hipLaunchKernelGGL((gated_norms_kernel<DT, W, NCH, true, true, USE>), grid, block, 0, stream, p);
    else if (p.post) hipLaunchKernelGGL((gated_norms_kernel<DT, W, NCH, true, false, USE>), grid, block, 0, stream, p);
    else if (p.q) hipLaunchKernelGGL((gated_norms_kernel<DT, W, NCH, false, true, USE>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gated_norms_kernel<DT, W, NCH, false, false, USE>), grid, block, 0, stream, p);
}

template <int DT, int W, int NCH>
void launch(const NormParams& p, hipStream_t stream) {
    const int64_t out = p.m * p.k * (p.q ? 3 : 4);
    if (out <= kL2Bytes) launch_use<DT, W, NCH, Use::Stores>(p, stream);
    else if (out <= kCacheBytes) launch_use<DT, W, NCH, Use::Plain>(p, stream);
    else launch_use<DT, W, NCH, Use::Both>(p, stream);
}

constexpr int64_t kMaxWidth = 16384;

// Waves of a row.  One wave holds up to 512 values in a chunk and joins nothing in LDS; four share wider rows.  From 513 to
// 1024 four waves leave up to half of themselves idle, which counts once the rows fill the chip (us, one wave / four, fp16
// out): 7188 x 64 5.9 / 12.5, 7188 x 512 6.8 / 13.1; 8 x 1024 4.1 / 3.6, 700 x 1024 4.4 / 4.2, 1024 x 1024 4.8 / 4.8, 1400 x 1024
// 5.0 / 5.5, 7188 x 1024 11.3 / 16.0, 7188 x 520 8.9 / 14.1; int8 rows 700 x 1024 4.7 / 4.6, 1024 x 1024 4.9 / 5.3, 7188 x 1024
// 12.3 / 17.9; 512 x 2048 6.2 / 4.4, 7188 x 2048 23.8 / 23.0.
constexpr int64_t kOneWaveRows = 1024;

template <int DT>
void dispatch(const NormParams& p, hipStream_t stream) {
    if (p.k <= 512) launch<DT, 1, 1>(p, stream);
    else if (p.k <= 1024 && p.m >= kOneWaveRows) launch<DT, 1, 2>(p, stream);
    else if (p.k <= 2048) launch<DT, 4, 1>(p, stream);
    else if (p.k <= 4096) launch<DT, 4, 2>(p, stream);
    else if (p.k <= 8192) launch<DT, 4, 4>(p, stream);
    else launch<DT, 4, 8>(p, stream);
}

int common(const char* what, int dtype, NormParams& p, int64_t gate_rows, int64_t k, hipStream_t stream) {
    H3V_REQUIRE(dtype == kF16 || dtype == kBF16, "%s: dtype must be 0 (fp16) or 1 (bf16)", what);
    H3V_REQUIRE(p.x && p.y && p.pre && p.h && (p.n || (p.q && p.scale)), "%s: null pointer argument", what);
    H3V_REQUIRE(p.m > 0 && p.m < (1 << 24), "%s: row count must be in [1, 2^24)", what);
    H3V_REQUIRE(k > 0 && k % 8 == 0 && k <= kMaxWidth, "%s: row width must be a multiple of 8 up to %lld (got %lld)", what,
                (long long)kMaxWidth, (long long)k);
    H3V_REQUIRE(p.eps > 0.0f && p.eps < 1.0f, "%s: epsilon must be in (0, 1)", what);
    H3V_REQUIRE(p.alpha - p.alpha == 0.0f, "%s: the residual scale must be finite", what);
    H3V_REQUIRE(!p.gate || (gate_rows > 0 && p.m % gate_rows == 0), "%s: gate rows must divide the row count", what);
    const void* const al[] = {p.x, p.y, p.gate, p.post, p.pre, p.h, p.n};
    for (const void* a : al) H3V_REQUIRE(aligned(a, 16), "%s: 16-bit pointers must be 16-byte aligned", what);
    H3V_REQUIRE(aligned(p.q, 8) && aligned(p.scale, 4), "%s: q must be 8-byte and scale 4-byte aligned", what);
    const int64_t e = p.m * k;
    H3V_REQUIRE(p.h + e <= p.y || p.y + e <= p.h, "%s: h must not overlap y", what);
    H3V_REQUIRE(p.h == p.x || p.h + e <= p.x || p.x + e <= p.h, "%s: h must be x or not overlap it", what);
    if (p.n)
        H3V_REQUIRE((p.n + e <= p.x || p.x + e <= p.n) && (p.n + e <= p.y || p.y + e <= p.n) && (p.n + e <= p.h || p.h + e <= p.n),
                    "%s: n must own separate storage", what);
    if (p.q) {
        auto apart = [&](const uint16_t* t) {
            const auto a = reinterpret_cast<uintptr_t>(p.q), b = reinterpret_cast<uintptr_t>(t);
            return a + e <= b || b + 2 * e <= a;
        };
        H3V_REQUIRE(apart(p.x) && apart(p.y) && apart(p.h), "%s: q must own separate storage", what);
    }
    p.k = (int)k;
    p.rows_per_gate = p.gate ? p.m / gate_rows : p.m;
    if (dtype == kF16) dispatch<kF16>(p, stream);
    else dispatch<kBF16>(p, stream);
    return launch_status(what);
}

}  // namespace
}  // namespace h3v

using namespace h3v;

extern "C" {

int h3v_gated_norms(int dtype, const uint16_t* x, const uint16_t* y, const uint16_t* gate, int64_t gate_rows,
                    const uint16_t* post, const uint16_t* pre, float alpha, float eps, int64_t m, int64_t k, uint16_t* h,
                    uint16_t* n, hipStream_t stream) {
    NormParams p = {x, y, gate, post, pre, alpha, eps, m, 0, 0, h, n, nullptr, nullptr};
    H3V_REQUIRE(n, "h3v_gated_norms: null pointer argument");
    return common("h3v_gated_norms", dtype, p, gate_rows, k, stream);
}

int h3v_gated_norms_quant(int dtype, const uint16_t* x, const uint16_t* y, const uint16_t* gate, int64_t gate_rows,
                          const uint16_t* post, const uint16_t* pre, float alpha, float eps, int64_t m, int64_t k,
                          uint16_t* h, int8_t* q, float* scale, hipStream_t stream) {
    NormParams p = {x, y, gate, post, pre, alpha, eps, m, 0, 0, h, nullptr, q, scale};
    return common("h3v_gated_norms_quant", dtype, p, gate_rows, k, stream);
}

}  // extern "C"
