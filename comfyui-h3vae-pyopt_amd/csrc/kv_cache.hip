// The INT8 K/V cache's write and read (layout and lookups: h3v_paged.hpp).
//
// Write.  A workgroup owns one (page, head) of keys or of values, so that a page's scale is settled by one workgroup:
//   a = max |x| over the page's new tokens,  s' = max(a * fl(1/127), 1e-30)
//   s = max(s_old, s') where the page holds earlier tokens, else s';  r = fl(1 / s)
//   new code = clamp(rint(fl(x * r)), -127, 127);  earlier code = rint(fl(code * fl(s_old / s))) where s moved
//   key mean = rint(fl(sum of the held codes / their count))
// An infinity or a NaN makes its page's scale that, and everything the page holds of the head reads as NaN until its
// first token is written again.  Places behind the last token keep what they hold.
//
// Read.  A workgroup owns one (page, head) of keys or values again; a value is fl(code * s) rounded once to 16 bits.
//
// Both are bound by memory, small calls by three latencies in a row (sequence, table, page): 4 x 1797 tokens of 32 heads of 64
// written in 23.5 us (88 MB) and read in 14.6; 64 single tokens of 8 heads of 128 written in 7.3 us, their pages read in 5.9.
#include "h3v_paged.hpp"

namespace h3v {
namespace {

struct WriteParams {
    Sequences s;
    const uint16_t* src[2];    // keys, values
    int64_t ts[2], hs[2];
    int8_t* codes[2];
    float* scale[2];
    int8_t* mean;
    int heads;
};

// The item-th touched page of the batch: sequence and logical page; false behind the last.
__device__ __forceinline__ bool touched_page(const Sequences& s, int page, int64_t item, int& b, int& j) {
    const int lane = threadIdx.x & 63;
    for (int at = 0; at < s.batch; at += 64) {
        int count = 0, first = 0;
        if (at + lane < s.batch) {
            const Span sp = span_of(s, at + lane);
            const int64_t cap = (int64_t)s.width * page;
            const int end = sp.len < cap ? sp.len : (int)cap;
            const int begin = sp.len > sp.n ? sp.len - sp.n : 0;
            first = begin / page;
            count = end > begin ? (end - 1) / page - first + 1 : 0;
        }
        int upto = count;   // inclusive prefix sum over the lanes
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off, 64);
            if (lane >= off) upto += v;
        }
        const int all = __shfl(upto, 63, 64);
        if (item < all) {
            const uint64_t m = __ballot(upto > item);
            const int l = __builtin_ctzll(m);
            b = at + l;
            j = __shfl(first, l, 64) + (int)item - (__shfl(upto, l, 64) - __shfl(count, l, 64));
            return true;
        }
        item -= all;
    }
    return false;
}

// A page of one head in units of 4 tokens x 8 dims.  The write gives a thread two of them (one: 26.6 us for 4 x 1797 tokens of 32
// heads of 64, two: 24.3, four: 24.1, but 4 us more for pages of 128 x 128), the read one; at most 256 threads.
constexpr int units_of(int dim, int page) { return page / 4 * (dim / 8); }
constexpr int threads_for(int units) { return units < 64 ? 64 : (units < 256 ? units : 256); }
constexpr int write_threads(int dim, int page) { return threads_for(units_of(dim, page) / 2); }
constexpr int read_threads(int dim, int page) { return threads_for(units_of(dim, page)); }

// four codes brought to another scale
__device__ __forceinline__ uint32_t moved_codes(uint32_t w, float ratio) {
    return codes4((float)(int8_t)w * ratio, (float)(int8_t)(w >> 8) * ratio, (float)(int8_t)(w >> 16) * ratio, (float)(int8_t)(w >> 24) * ratio);
}

template <int DT, int D, int P>
__global__ __launch_bounds__(write_threads(D, P)) void kv_write_kernel(WriteParams p) {
    constexpr int NT = write_threads(D, P), NU = units_of(D, P) / NT, NWV = NT / 64;
    constexpr int LD = D / 8;                           // lanes of a token row
    constexpr int kRow = P / 4 + 1;                     // words of a dim's tokens in LDS, one of padding
    __shared__ uint32_t tile[D * kRow];
    __shared__ uint32_t red[NWV];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // neighbours take the heads of one page: together they read whole token rows
    const int which = blockIdx.z, head = blockIdx.x % p.heads;
    int b, j;
    if (!touched_page(p.s, P, blockIdx.x / p.heads, b, j)) return;
    b = __builtin_amdgcn_readfirstlane(b);
    j = __builtin_amdgcn_readfirstlane(j);
    const Span sp = span_of(p.s, b);
    const int id = page_id(p.s, b, j);
    const int shift = sp.len - sp.n;                    // position of packed row sp.row (negative: not there)
    const int lo = j * P;
    const int begin = max(shift, lo) - lo, end = min(sp.len - lo, P);   // new tokens of the page
    const uint16_t* const src = p.src[which] + (sp.row + lo - shift) * p.ts[which] + head * p.hs[which];
    const int dch = tid % LD, tg0 = tid / LD;
    // tokens of a unit: for keys a quarter page apart, so that a wave writes whole rows side by side; for values four in a
    // row, a word of the transposed page
    const int step = which == 0 ? P / 4 : 1, first = which == 0 ? 1 : 4;

    // every load of the page before the first use of one
    u32x4 x[NU][4];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = (tg0 + u * (NT / LD)) * first + i * step;
            x[u][i] = u32x4{0, 0, 0, 0};
            if (t >= begin && t < end) x[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + t * p.ts[which] + 8 * dch));
        }
    if (id < 0) return;
    const int64_t ph = (int64_t)id * p.heads + head;
    int8_t* const codes = p.codes[which] + ph * (P * D);
    float s_old = 0.0f;
    uint2 old[NU][4] = {};
    if (begin > 0) {
        s_old = p.scale[which][ph];
        if (which == 0) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = tg0 + u * (NT / LD) + i * (P / 4);
                    if (t < begin) old[u][i] = *reinterpret_cast<const uint2*>(codes + t * D + 8 * dch);
                }
        }
    }
    u16x2 tops = {0, 0};
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) tops = max_magnitudes(tops, x[u][i][w]);
    uint32_t top = max(tops[0], tops[1]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    if constexpr (NWV > 1) {
        if (lane == 0) red[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NWV; ++w) top = max(top, red[w]);
    }
    const float s_new = code_scale(to_f32<DT>((uint16_t)top));
    float s = s_new, ratio = 1.0f;
    bool moved = false;
    if (begin > 0) {
        s = (s_old != s_old || s_old > s_new) ? s_old : s_new;
        moved = s != s_old;
        ratio = s_old / s;
    }
    const float r = 1.0f / s;
    if (tid == 0) p.scale[which][ph] = s;

    if (which == 0) {
        // sums of the dims 0 and 2, 1 and 3, 4 and 6, 5 and 7 of the lane's 8, two 16-bit sums per word (at most 128 * 127)
        s16x2 sum[4] = {};
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = tg0 + u * (NT / LD) + i * (P / 4);
                if (t >= end) continue;
                uint32_t q[2] = {old[u][i].x, old[u][i].y};
                if (t >= begin) {
                    float v[8];
                    unpack8<DT>(x[u][i], v);
                    q[0] = codes4(v[0] * r, v[1] * r, v[2] * r, v[3] * r);
                    q[1] = codes4(v[4] * r, v[5] * r, v[6] * r, v[7] * r);
                } else if (moved) {
#pragma unroll
                    for (int w = 0; w < 2; ++w) q[w] = moved_codes(q[w], ratio);
                }
                if (t >= begin || moved) *reinterpret_cast<uint2*>(codes + t * D + 8 * dch) = make_uint2(q[0], q[1]);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    sum[2 * w] += __builtin_bit_cast(s16x2, q[w] << 8) >> 8;
                    sum[2 * w + 1] += __builtin_bit_cast(s16x2, q[w]) >> 8;
                }
            }
        // first the lanes of a wave that hold the same dims, then the waves
        int* const part = reinterpret_cast<int*>(tile);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int off = LD; off < 64; off <<= 1) sum[e] += __builtin_bit_cast(s16x2, __shfl_xor(__builtin_bit_cast(int, sum[e]), off, 64));
            if (lane < LD) part[wave * (D / 2) + 4 * lane + e] = __builtin_bit_cast(int, sum[e]);
        }
        __syncthreads();   // also where one wave is the workgroup: its lanes read what other lanes wrote
        if (tid < D / 4) {
            s16x2 a = {0, 0}, c = {0, 0};      // dims 4 tid and + 2, + 1 and + 3
#pragma unroll
            for (int w = 0; w < NWV; ++w) {
                a += __builtin_bit_cast(s16x2, part[w * (D / 2) + 2 * tid]);
                c += __builtin_bit_cast(s16x2, part[w * (D / 2) + 2 * tid + 1]);
            }
            const float held = (float)end;
            reinterpret_cast<uint32_t*>(p.mean + ph * D)[tid] =
                codes4((float)a[0] / held, (float)c[0] / held, (float)a[1] / held, (float)c[1] / held);
        }
    } else {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            float v[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack8<DT>(x[u][i], v[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                tile[(8 * dch + e) * kRow + tg0 + u * (NT / LD)] =
                    codes4(v[0][e] * r, v[1][e] * r, v[2][e] * r, v[3][e] * r);
        }
        __syncthreads();
        if (begin == 0 && end == P) {
            for (int w = tid; w < D * (P / 16); w += NT) {
                const uint32_t* const from = tile + w / (P / 16) * kRow + w % (P / 16) * 4;
                *reinterpret_cast<u32x4*>(codes + 16 * w) = u32x4{from[0], from[1], from[2], from[3]};
            }
            return;
        }
        // a page that is begun or not full: the words that hold a token whose code changes, four of a thread in flight
        const int w0 = moved ? 0 : begin >> 2, nw = ((end - 1) >> 2) - w0 + 1;
        for (int base = tid; base < D * nw; base += 4 * NT) {
            uint32_t* at[4];
            uint32_t was[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int w = base + i * NT, d = w / nw, tg = w0 + w % nw;
                at[i] = reinterpret_cast<uint32_t*>(codes + d * P) + tg;
                was[i] = w < D * nw ? *at[i] : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int w = base + i * NT, d = w / nw, tg = w0 + w % nw;
                if (w >= D * nw) continue;
                const uint32_t now = tile[d * kRow + tg];
                uint32_t out = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 4 * tg + e;
                    int q = (int8_t)((t >= begin && t < end ? now : was[i]) >> (8 * e));
                    if (t < begin && moved) q = code8((float)q * ratio);
                    out |= (uint32_t)(q & 0xff) << (8 * e);
                }
                *at[i] = out;
            }
        }
    }
}

// A read's outputs are stored past the L2s where they fit there with room for a reader's own, so that none are left to write back at
// the kernel's end, and where they are more than the Infinity Cache holds; between, they are left there for their reader. us, plain /
// streamed, alone and with a sum that reads them: 12 MB 5.6 / 4.7, 12.9 / 12.2; 17 MB 7.1 / 5.7, 15.7 / 14.8; 20.5 MB 7.5 / 5.3, 17.2 /
// 17.1; 24 MB 8.3 / 5.8, 18.2 / 18.8; 31 MB 9.3 / 8.4, 18.7 / 20.1; 59 MB 15.6 / 15.6, 29.3 / 30.7; 197 MB 48 / 45, 94 / 105; 328 MB
// 97 / 91, 182 / 177; 655 MB 191 / 179, 358 / 350.
constexpr int64_t kStreamBelow = 20 << 20, kStreamAbove = 256 << 20;

struct ReadParams {
    Sequences s;
    const int* first;
    const int8_t* codes[2];
    const float* scale[2];
    uint16_t* out[2];
    int heads, length;
};

// STREAM: outputs are stored past the L2s.
template <int DT, int D, int P, bool STREAM>
__global__ __launch_bounds__(read_threads(D, P)) void kv_read_kernel(ReadParams p) {
    constexpr int NT = read_threads(D, P), NU = units_of(D, P) / NT;
    constexpr int LD = D / 8;
    constexpr int kRow = P / 4 + 1;
    constexpr int NW = D * P / 16 / NT;                 // 16-byte loads of a page per thread
    __shared__ uint32_t tile[D * kRow];
    const int tid = threadIdx.x;
    const int which = blockIdx.z & 1, b = blockIdx.z >> 1, head = blockIdx.x % p.heads;
    const int64_t first = p.first[b], held_all = p.s.lens[b];
    // tokens of the output that lie in page j: floor division, so that a negative first is only rows that are not there
    const int64_t base = first >= 0 ? first / P : -((P - 1 - first) / P);
    const int64_t j = base + blockIdx.x / p.heads;
    const int64_t t0 = j * P - first;                   // output row of the page's first token
    if (t0 >= p.length) return;
    const int64_t len = min(held_all, (int64_t)p.s.width * P);
    const int id = j >= 0 && j * P < len ? page_id(p.s, b, (int)j) : -1;
    const int held = id < 0 ? 0 : (int)min(len - j * P, (int64_t)P);
    const int64_t ph = (int64_t)max(id, 0) * p.heads + head;
    const int8_t* const codes = p.codes[which] + ph * (P * D);
    const int dch = tid % LD, tg0 = tid / LD;
    uint16_t* const out = p.out[which] + (((int64_t)b * p.length + t0) * p.heads + head) * D + 8 * dch;
    const int64_t row = (int64_t)p.heads * D;
    float s = 0.0f;
    uint2 w[NU][4] = {};                                // keys: 8 codes of tokens a quarter page apart
    if (held > 0) {
        s = p.scale[which][ph];
        if (which == 0) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[u][i] = *reinterpret_cast<const uint2*>(codes + (tg0 + u * (NT / LD) + i * (P / 4)) * D + 8 * dch);
        } else {
            u32x4 v[NW];
#pragma unroll
            for (int i = 0; i < NW; ++i) v[i] = *reinterpret_cast<const u32x4*>(codes + 16 * (tid + i * NT));
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int c = tid + i * NT;
                uint32_t* const to = tile + c / (P / 16) * kRow + c % (P / 16) * 4;
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = v[i][e];
            }
        }
    }
    // eight values of token t, code(e) of dim 8 dch + e
    auto put = [&](int t, auto&& code) {
        if (t0 + t < 0 || t0 + t >= p.length) return;
        const float st = t < held ? s : 0.0f;            // with the codes behind the last token made zeros
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)code(e) * st;
        if constexpr (STREAM) __builtin_nontemporal_store(pack8<DT>(v), reinterpret_cast<u32x4*>(out + t * row));
        else *reinterpret_cast<u32x4*>(out + t * row) = pack8<DT>(v);
    };
    if (which == 0) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = tg0 + u * (NT / LD) + i * (P / 4);
                const uint32_t lo = t < held ? w[u][i].x : 0u, hi = t < held ? w[u][i].y : 0u;
                put(t, [&](int e) { return (int8_t)((e < 4 ? lo : hi) >> (8 * (e & 3))); });
            }
        return;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int tg = tg0 + u * (NT / LD), left = held - 4 * tg;       // tokens of the word that are held
        const uint32_t mask = left >= 4 ? ~0u : (left <= 0 ? 0u : (1u << (8 * left)) - 1u);
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = held > 0 ? tile[(8 * dch + e) * kRow + tg] & mask : 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            put(4 * tg + i, [&](int e) { return (int8_t)(c[e] >> (8 * i)); });
    }
}

}  // namespace
}  // namespace h3v

using namespace h3v;

extern "C" {

int h3v_kv_cache_write(int dtype, const uint16_t* k, int64_t k_token_stride, int64_t k_head_stride, const uint16_t* v,
                       int64_t v_token_stride, int64_t v_head_stride, int64_t tokens, const int* starts, const int* lens,
                       const int* table, int64_t batch, int64_t width, int64_t heads, int64_t dim, int64_t page,
                       int64_t pages, int8_t* k_cache, int8_t* v_cache, float* k_scale, float* v_scale, int8_t* k_mean,
                       hipStream_t stream) {
    const char* what = "h3v_kv_cache_write";
    H3V_REQUIRE(batch > 0 && batch <= 32768 && width > 0 && width <= (1 << 23), "%s: batch or table width out of range", what);
    const Sequences s = {starts, lens, table, (int)batch, (int)width, tokens, pages};
    const int rc = check_paged(what, dtype, s, heads, dim, page);
    if (rc) return rc;
    H3V_REQUIRE(k && v && starts && k_cache && v_cache && k_scale && v_scale && k_mean, "%s: null pointer argument", what);
    H3V_REQUIRE(tokens > 0 && tokens <= (1 << 27), "%s: tokens must be in [1, 2^27]", what);
    const int64_t strides[4] = {k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    for (int64_t st : strides)
        H3V_REQUIRE(st > 0 && st % 8 == 0, "%s: token/head strides must be positive multiples of 8 elements (16-byte rows)", what);
    H3V_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(k_mean, 16),
                "%s: k, v and the cache must be 16-byte aligned", what);
    H3V_REQUIRE(aligned(k_scale, 4) && aligned(v_scale, 4), "%s: scales must be 4-byte aligned", what);
    WriteParams p = {s, {k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, {k_cache, v_cache},
                     {k_scale, v_scale}, k_mean, (int)heads};
    // a sequence of n new tokens touches at most min(n, n / page + 2) pages
    const int64_t items = tokens < tokens / page + 2 * batch ? tokens : tokens / page + 2 * batch;
    H3V_REQUIRE(items * heads * 256 <= 0xffffffffll, "%s: too many pages of new tokens", what);
    const dim3 grid((unsigned)(items * heads), 1, 2);
    by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
        hipLaunchKernelGGL((kv_write_kernel<dt(), d(), pg()>), grid, dim3(write_threads(d(), pg())), 0, stream, p);
    });
    return launch_status(what);
}

int h3v_kv_cache_read(int dtype, const int8_t* k_cache, const int8_t* v_cache, const float* k_scale, const float* v_scale,
                      const int* first, const int* lens, const int* table, int64_t batch, int64_t width, int64_t length,
                      int64_t heads, int64_t dim, int64_t page, int64_t pages, uint16_t* k, uint16_t* v,
                      hipStream_t stream) {
    const char* what = "h3v_kv_cache_read";
    H3V_REQUIRE(batch > 0 && batch <= 32767 && width > 0 && width <= (1 << 23), "%s: batch or table width out of range", what);
    const Sequences s = {nullptr, lens, table, (int)batch, (int)width, 0, pages};
    const int rc = check_paged(what, dtype, s, heads, dim, page);
    if (rc) return rc;
    H3V_REQUIRE(k_cache && v_cache && k_scale && v_scale && first && k && v, "%s: null pointer argument", what);
    H3V_REQUIRE(length > 0 && length <= (1 << 27), "%s: length must be in [1, 2^27]", what);
    H3V_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(first, 4) &&
                    aligned(k_scale, 4) && aligned(v_scale, 4),
                "%s: outputs and cache must be 16-byte, the others 4-byte aligned", what);
    ReadParams p = {s, first, {k_cache, v_cache}, {k_scale, v_scale}, {k, v}, (int)heads, (int)length};
    const int64_t tiles = (length / page + 2) * heads;
    H3V_REQUIRE(tiles * 256 <= 0xffffffffll, "%s: too long", what);
    const dim3 grid((unsigned)tiles, 1, (unsigned)(2 * batch));
    const int64_t bytes = 4 * batch * length * heads * dim;
    const bool stream_out = bytes <= kStreamBelow || bytes > kStreamAbove;
    by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
        if (stream_out) hipLaunchKernelGGL((kv_read_kernel<dt(), d(), pg(), true>), grid, dim3(read_threads(d(), pg())), 0, stream, p);
        else hipLaunchKernelGGL((kv_read_kernel<dt(), d(), pg(), false>), grid, dim3(read_threads(d(), pg())), 0, stream, p);
    });
    return launch_status(what);
}

}  // extern "C"
