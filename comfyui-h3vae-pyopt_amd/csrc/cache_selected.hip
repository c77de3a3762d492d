// Attention over selected pages for several new tokens per sequence (one token per sequence: cache_attention.hip, the same
// operator with a list).
//
// Tokens next to each other mostly select the same pages.  A workgroup takes as many consecutive tokens of a sequence
// as the 16 rows of a tile hold heads of (16 / columns, columns the group's size as a power of two) and walks the union
// of their lists, ascending; a mask per page says which tokens it is for, and the rows of the others see none of its
// keys.  At worst, with lists that share nothing, that is the work of a token at a time.  The union is made in LDS: a
// mask per page of the sequence, then one scan that lists the pages that have one.  A list that names a page twice
// counts it twice: such tiles (found while the masks are made) walk each token's own list instead.
//
// 2048 tokens over 16384, 16 heads on 4 kv heads of 64, 32 pages of 64 each: 117 us, 142 with the selection (217 a token at
// a time), bound by instructions: vector units 87%, matrix units 18% of the time.
#include "cache_rows.hpp"

namespace h3v {
namespace {

constexpr int kNW = 4;
constexpr int kNT = 64 * kNW;

struct SelectedParams {
    AttnParams a;
    int columns, tile;     // rows of a token (a power of two), tokens of a tile
    int row;               // pages that the masks cover, a multiple of kNT
};

template <int DT, int D, int P>
__global__ __launch_bounds__(kNT, D == 64 ? 3 : 2) void cache_selected_kernel(SelectedParams q) {
    using Tile = RowTile<DT, D, P>;
    // masks [row] of 16 bits, then the list: pages [capacity] and their masks; the joined parts reuse the place
    extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
    __shared__ int scan[kNW], twice;
    const AttnParams& p = q.a;
    uint32_t* const masks = lds;
    uint32_t* const list = lds + q.row / 2;
    Joined<D, kNW>& joined = *reinterpret_cast<Joined<D, kNW>*>(lds);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15;
    const int64_t t0 = (int64_t)blockIdx.x * q.tile;
    const int kvh = blockIdx.y;
    const int tokens = (int)min((int64_t)q.tile, p.s.tokens - t0);
    const int mine = col / q.columns, head = col % q.columns;
    const bool real = mine < tokens && head < p.group;

    Tile rt;
    rt.load_rows(p.q + (t0 + (real ? mine : 0)) * p.q_ts + (int64_t)(kvh * p.group + (real ? head : 0)) * p.q_hs);
    rt.set_rows(p.c);

    // runs of the tile's tokens that belong to one sequence
    for (int c0 = 0; c0 < tokens;) {
        const int b = __builtin_amdgcn_readfirstlane(sequence_of(p.s, t0 + c0));
        int c1 = c0 + 1, seen = 0, last = 0;
        if (b >= 0) {
            const Span sp = span_of(p.s, b);
            c1 = (int)min((int64_t)tokens, max((int64_t)c1, sp.row + sp.n - t0));
            const int first = (int)(t0 - sp.row);             // the tile's first token in the sequence
            if (real && mine >= c0 && mine < c1) seen = keys_seen(p, sp, first + mine, P);
            last = keys_seen(p, sp, first + c1 - 1, P);
        }
        const int pages = (last + P - 1) / P;                 // at most the table's width
        rt.reset();

        // the union of the run's lists
        for (int i = tid; i < (pages + 1) / 2; i += kNT) masks[i] = 0;
        if (tid == 0) twice = 0;
        __syncthreads();
        const int* const sel = p.sel + ((t0 + c0) * p.kv_heads + kvh) * p.blocks;
        for (int i = tid; i < (c1 - c0) * p.blocks; i += kNT) {
            const int c = i / p.blocks, j = sel[(int64_t)c * p.kv_heads * p.blocks + i % p.blocks];
            if (j < 0 || j >= pages) continue;
            const uint32_t bit = 1u << (c0 + c + 16 * (j & 1));
            if (atomicOr(&masks[j >> 1], bit) & bit) twice = 1;
        }
        __syncthreads();
        const bool apart = twice != 0;
        for (int c = c0; c < (apart ? c1 : c0 + 1); ++c) {
            int entries;
            if (!apart) {
                // a thread looks at a run of consecutive pages
                const int run = (pages + kNT - 1) / kNT, j0 = min(tid * run, pages), j1 = min(j0 + run, pages);
                int n = 0;
                for (int j = j0; j < j1; ++j) n += (masks[j >> 1] >> (16 * (j & 1)) & 0xffffu) != 0;
                int upto = n;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const int v = __shfl_up(upto, off, 64);
                    if (lane >= off) upto += v;
                }
                if (lane == 63) scan[wave] = upto;
                __syncthreads();
                entries = 0;
                int at = upto - n;
#pragma unroll
                for (int w = 0; w < kNW; ++w) {
                    if (w < wave) at += scan[w];
                    entries += scan[w];
                }
                for (int j = j0; j < j1; ++j) {
                    const uint32_t m = masks[j >> 1] >> (16 * (j & 1)) & 0xffffu;
                    if (m) list[at++] = (uint32_t)j | m << 16;
                }
            } else {
                entries = p.blocks;
                for (int i = tid; i < p.blocks; i += kNT) {
                    const int j = sel[(int64_t)(c - c0) * p.kv_heads * p.blocks + i];
                    list[i] = j < 0 || j >= pages ? 0u : (uint32_t)j | 0x10000u << c;   // no token: passed over
                }
            }
            __syncthreads();
            // the wave's entries wave, + kNW, ...: 64 at a time, page, mask, id and scales one per lane
            for (int jb = wave; jb < entries; jb += 64 * kNW) {
                uint32_t my = 0;
                int my_id = -1;
                float my_ks = 0.0f, my_vs = 0.0f;
                if (jb + lane * kNW < entries) {
                    my = list[jb + lane * kNW];
                    if (my >> 16) my_id = page_id(p.s, b, (int)(my & 0xffffu));
                }
                if (my_id >= 0) {
                    my_ks = p.ks[(int64_t)my_id * p.kv_heads + kvh];
                    my_vs = p.vs[(int64_t)my_id * p.kv_heads + kvh] * (1.0f / (1 << kOutDrop));
                }
                struct Step {
                    typename Tile::Codes codes;
                    int lane, sub;
                };
                uint64_t left = __ballot(my_id >= 0);
                int sub = 0;
                Tile::template run<Step>(
                    __popcll(left) * Tile::NSUB,
                    [&](Step& w) {
                        w.lane = __builtin_ctzll(left);
                        w.sub = sub;
                        const int id = __builtin_amdgcn_readlane(my_id, w.lane);
                        rt.template load<false>(w.codes, p.k, p.v, (int64_t)id * p.kv_heads + kvh, sub);
                        if (++sub == Tile::NSUB) {
                            sub = 0;
                            left &= left - 1;
                        }
                    },
                    [&](Step& w) {
                        const uint32_t e = __builtin_amdgcn_readlane(my, w.lane);
                        const int key0 = (int)(e & 0xffffu) * P + w.sub * Tile::KT;
                        if (Tile::NSUB > 1 && key0 >= last) return;
                        rt.attend(w.codes, key0, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_ks), w.lane)),
                                  __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_vs), w.lane)),
                                  e >> (16 + mine) & 1 ? seen : 0);
                    });
            }
            __syncthreads();   // the list is read
        }

        joined.put(rt, wave);
        __syncthreads();
        for (int e = tid; e < 16 * (D / 4); e += kNT) {
            const int r = e / (D / 4), d = e % (D / 4) * 4, c = r / q.columns, h = r % q.columns;
            if (c < c0 || c >= c1 || h >= p.group) continue;
            float top, sum;
            const f32x4 out = joined.get(r, d, top, sum);
            put_row<DT>(p.o + ((t0 + c) * p.heads + kvh * p.group + h) * D + d, out, row_inverse(top, sum));
        }
        __syncthreads();   // the parts are read
        c0 = c1;
    }
}

}  // namespace

int selected_tile(int64_t tokens, int64_t batch, int64_t width, int64_t group, int64_t blocks) {
    // At a token or less per sequence the tokens next to each other are strangers.  Pages are listed in 16 bits, and
    // masks (2 bytes a page) and list (at most the pages, or the tile's entries) share 128 KB.
    if (tokens <= batch || width > 32768) return 1;
    int64_t columns = 1, tile = 1;
    while (columns < group) columns *= 2;
    while (2 * tile * columns <= 16 && 2 * tile * blocks <= 16384) tile *= 2;
    return (int)tile;
}

int launch_selected(const char* what, const AttnParams& p, int tile, int dtype, int64_t dim, int64_t page, hipStream_t stream) {
    SelectedParams q = {p, 1, tile, (p.s.width + kNT - 1) / kNT * kNT};
    while (q.columns < p.group) q.columns *= 2;
    const int64_t list = tile * p.blocks < q.row ? tile * p.blocks : q.row;
    const int64_t words = q.row / 2 + (list > p.blocks ? list : p.blocks), joined = kNW * 16 * (dim + 4 + 2);
    const unsigned lds = (unsigned)(4 * (words > joined ? words : joined));
    const dim3 grid((unsigned)((p.s.tokens + tile - 1) / tile), (unsigned)p.kv_heads);
    int rc = H3V_OK;
    by_shape(dtype, dim, page, [&](auto dt, auto d, auto pg) {
        rc = reserve_lds<cache_selected_kernel<dt(), d(), pg()>>(what, 150 << 10);
        if (rc) return;
        hipLaunchKernelGGL((cache_selected_kernel<dt(), d(), pg()>), grid, dim3(kNT), lds, stream, q);
    });
    return rc;
}

}  // namespace h3v
