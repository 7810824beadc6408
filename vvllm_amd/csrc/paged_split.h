// Attention of one query per sequence over a paged cache, whatever its rows hold: a tile of up to 16 query heads of one kv
// head is a wave's work on a chunk of keys, and here is how a batch's tiles and chunks are shared out and joined.  A class TL
// of static members says the rest: Args (the cache; B, P, max_pages), T (queries and outputs), D, CH (keys of a chunk), HEAD
// (chunks that the beginning of a tile is as long as: what comes before the first chunk's products counts in a batch of
// short contexts), COLUMNS (a head's sums may be in several columns: put, store and join write what this code writes for the
// others, whose outputs keep the divisions and exponentials that they always had, to the last bit), VB (bytes of LDS a wave),
// Q (a tile's queries in registers), load_q, tile (the chunks c0, c0 + cstep, ... below ke of sequence s and kv head g), dim
// (of accumulator element (e, lane group, i)).
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// Head (lane % 16)'s running maximum, sum and output fragments: o[e][i] is dim
// TL::dim(e, lane / 16, i).
template <int D>
struct PagedAcc {
    float m, l;
    f4 o[D / 16];
    __device__ __forceinline__ void clear()
    {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < D / 16; e++) o[e] = f4{};
    }
};

// Sequence s's length, as the kernels take it
template <typename Args>
__device__ __forceinline__ int32_t paged_len(const Args& c, const int32_t* lens, int32_t s)
{
    const int64_t cap = (int64_t)c.max_pages * c.P;
    const int32_t n = lens[s];
    return n < 0 ? 0 : n < cap ? n : (int32_t)cap;
}

// What tile v of a sequence is: its kv head, first query head and number of heads.
struct PagedHeads {
    int32_t G, GT, tiles;  // heads of a kv head, of a tile, tiles of a kv head
    __device__ __forceinline__ void at(int32_t v, int32_t& g, int32_t& h0, int32_t& n) const
    {
        g = v / tiles;
        const int32_t t = v - g * tiles;
        h0 = g * G + t * GT;
        n = G - t * GT < GT ? G - t * GT : GT;
    }
};

// One tile of one sequence by one block, its NW waves each every NW-th chunk, merged through LDS.
template <typename TL, int NW>
__device__ __forceinline__ void paged_one(const typename TL::Args& c, typename TL::T* __restrict__ out,
                                          const typename TL::T* __restrict__ q, const int32_t* __restrict__ lens, PagedHeads hd,
                                          int32_t H, float scale_log2)
{
    constexpr int D = TL::D, CH = TL::CH, OP = D + 4;
    constexpr int VB = TL::VB, OB = 16 * OP * 4;  // bytes a wave
    __shared__ __align__(16) char smem[NW * (VB > OB ? VB : OB)];
    __shared__ float wm[NW][16], wl[NW][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, gr = lane >> 4;
    const int32_t s = blockIdx.y, len = paged_len(c, lens, s);
    int32_t g, h0, n;
    hd.at(blockIdx.x, g, h0, n);
    const int64_t row0 = (int64_t)s * H + h0;
    typename TL::Q x;
    TL::load_q(q + row0 * D, n, lane, x);
    PagedAcc<D> acc;
    TL::tile(c, g, s, x, w * CH, NW * CH, len, scale_log2, smem + w * VB, lane, acc);
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);
    if (gr == 0) {
        wm[w][r] = acc.m;
        wl[w][r] = acc.l;
    }
#pragma unroll
    for (int e = 0; e < D / 16; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) os[(w * 16 + r) * OP + TL::dim(e, gr, i)] = acc.o[e][i];
    __syncthreads();
    for (int idx = threadIdx.x; idx < n * D; idx += 64 * NW) {
        const int h = idx / D, d = idx - h * D;
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < NW; i++) M = fmaxf(M, wm[i][h]);
        const float Mb = M == -INFINITY ? 0.0f : M;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; i++) attn_merge_add(num, den, wm[i][h], Mb, os[(i * 16 + h) * OP + d], wl[i][h]);
        out[row0 * D + idx] = (typename TL::T)(den == 0.0f ? 0.0f : num / den);
    }
}

// Units of the 64 sequences from s0 on, one a lane, and their sums up to each lane: a sequence's chunks, and TL::HEAD for
// the beginning of a tile, where there is any.
template <typename TL>
__device__ __forceinline__ int32_t paged_window(const typename TL::Args& c, const int32_t* lens, int32_t s0, int lane)
{
    const int32_t n = s0 + lane < c.B ? (paged_len(c, lens, s0 + lane) + TL::CH - 1) / TL::CH : 0;
    return n > 0 ? n + TL::HEAD : 0;
}
// Sums over lanes 0 .. l in lane l (shifts within rows of 16, then the rows' last lanes broadcast).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ int64_t lane_of64(uint64_t v, int l)
{
    return (int64_t)((uint64_t)lane_of((uint32_t)(v >> 32), l) << 32 | lane_of((uint32_t)v, l));
}

// a b / c and a / c, in 32 bits where they fit (a 64-bit division is 100 instructions)
__device__ __forceinline__ uint64_t muldiv(uint64_t a, uint64_t b, uint64_t c)
{
    const uint64_t p = a * b;
    return (p | c) >> 32 ? p / c : (uint32_t)p / (uint32_t)c;
}

// All chunks of all tiles of all sequences in one row (sequence by sequence, tile by
// tile): wave w of W (all waves, or T) takes units [T w / W, T (w + 1) / W) of its T, so
// every wave has the same work however ragged the batch.  The part of a tile that a wave has goes
// straight to out if it is the whole tile, else to the wave's slot 1 (a tile that
// begins in its range) or 0, a row per head: O, m, l.  Where all four waves of a block are in one tile,
// their parts are added through LDS and go to the first one's slot.  k_attention_paged_merge joins what there is.
template <typename TL>
__device__ __forceinline__ void paged_split(const typename TL::Args& c, typename TL::T* __restrict__ out,
                                            const typename TL::T* __restrict__ q, const int32_t* __restrict__ lens, PagedHeads hd,
                                            int32_t H, float scale_log2, int64_t* __restrict__ before_out, float* __restrict__ ws,
                                            int32_t VH)
{
    constexpr int D = TL::D, CH = TL::CH;
    constexpr int VB = TL::VB, OP = D + 4, OB = 16 * OP * 4;  // bytes a wave
    __shared__ __align__(16) char smem[4 * (VB > OB ? VB : OB)];
    __shared__ float wm[4][16], wl[4][16];
    const int lane = threadIdx.x & 63, r = lane & 15, gr = lane >> 4;
    const int wb = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = (int64_t)blockIdx.x * 4 + wb;
    // the sums of the chunks before each sequence, and of all: the first wave keeps them for the merge
    int64_t total = 0;
    int32_t n = 0;  // the first 64 sequences' units, and their sums
    uint32_t upto = 0;
    for (int32_t s0 = 0; s0 < c.B; s0 += 64) {
        const int32_t m = paged_window<TL>(c, lens, s0, lane);
        const uint32_t sums = wave_scan((uint32_t)m);  // at most 64 * 2^25
        if (s0 == 0) {
            n = m;
            upto = sums;
        }
        if (w == 0 && s0 + lane < c.B) before_out[s0 + lane + 1] = total + sums;
        total += lane_of(sums, 63);
    }
    if (w == 0 && lane == 0) before_out[0] = 0;
    total *= VH;
    const int64_t W = total < (int64_t)gridDim.x * 4 ? total : (int64_t)gridDim.x * 4;  // no wave without a unit
    if (w >= W) return;
    // lane l: where wave l of the block begins, and the next block (l = 4)
    const uint64_t begin = muldiv(total, w - wb + (lane < 4 ? lane : 4), W);
    auto begin_of = [&](int l) { return lane_of64(begin, l); };
    const int64_t u0 = begin_of(wb), u1 = begin_of(wb + 1);
    // the window of sequences that holds unit u0
    int32_t s0 = 0;
    int64_t before = 0;
    while ((before + lane_of(upto, 63)) * VH <= u0) {
        before += lane_of(upto, 63);
        s0 += 64;
        n = paged_window<TL>(c, lens, s0, lane);
        upto = wave_scan((uint32_t)n);
    }
    int sl = __builtin_ctzll(__ballot((before + upto) * VH > u0));  // the sequence's lane
    int32_t ns = (int32_t)lane_of((uint32_t)n, sl);
    const int64_t rest = u0 - (before + lane_of(upto, sl) - ns) * VH;  // units before u0 in the sequence
    int32_t v = __builtin_amdgcn_readfirstlane((int32_t)muldiv(rest, 1, ns));
    int32_t ci = __builtin_amdgcn_readfirstlane((int32_t)(rest - (int64_t)v * ns));
    // the block's range within this wave's first tile
    const int64_t b0 = begin_of(0), b1 = begin_of(4);
    const bool inside = w - wb + 4 <= W && u0 - b0 <= ci && b1 - u0 <= ns - ci;
    for (int64_t u = u0; u < u1;) {
        const int32_t s = s0 + sl, cnt = (int32_t)(ns - ci < u1 - u ? ns - ci : u1 - u);
        int32_t g, h0, nh;
        hd.at(v, g, h0, nh);
        const int64_t row0 = (int64_t)s * H + h0;
        typename TL::Q x;
        TL::load_q(q + row0 * D, nh, lane, x);
        PagedAcc<D> acc;
        const int32_t len = __builtin_amdgcn_readfirstlane(paged_len(c, lens, s));
        const int32_t first = ci > TL::HEAD ? ci - TL::HEAD : 0;  // chunk; a range of the tile's head alone has none
        const int64_t end = (int64_t)(ci + cnt - TL::HEAD) * CH;
        TL::tile(c, g, s, x, first * CH, CH, end < len ? (int32_t)end : len, scale_log2, smem + wb * VB, lane, acc);
        if constexpr (TL::COLUMNS) {
            const bool whole = inside ? b1 - b0 == ns : cnt == ns;
            if (inside) {
                __syncthreads();
                float* os = reinterpret_cast<float*>(smem);
                TL::put(acc, lane, nh, os + wb * 16 * OP, OP, wm[wb], wl[wb]);
                __syncthreads();
                float* part = ws + ((w - wb) * 2 + (u0 - b0 == ci)) * hd.GT * (D + 4);
                TL::template join<4>(whole ? out + row0 * D : nullptr, part, wm, wl, os, nh);
                return;
            }
            if (whole) TL::store(acc, lane, nh, out + row0 * D);
            else TL::put(acc, lane, nh, ws + (w * 2 + (ci == 0)) * hd.GT * (D + 4), D + 4, nullptr, nullptr);
        } else {
            if (inside) {
                __syncthreads();
                float* os = reinterpret_cast<float*>(smem);
                if (gr == 0) {
                    wm[wb][r] = acc.m;
                    wl[wb][r] = acc.l;
                }
#pragma unroll
                for (int e = 0; e < D / 16; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) os[(wb * 16 + r) * OP + TL::dim(e, gr, i)] = acc.o[e][i];
                __syncthreads();
                const bool whole = b1 - b0 == ns;
                float* part = ws + ((w - wb) * 2 + (u0 - b0 == ci)) * hd.GT * (D + 4);
                for (int idx = threadIdx.x; idx < nh * D; idx += 256) {
                    const int h = idx / D, d = idx - h * D;
                    const float M = fmaxf(fmaxf(wm[0][h], wm[1][h]), fmaxf(wm[2][h], wm[3][h])), Mb = M == -INFINITY ? 0.0f : M;
                    float num = 0.0f, den = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; i++) attn_merge_add(num, den, wm[i][h], Mb, os[(i * 16 + h) * OP + d], wl[i][h]);
                    if (whole) {
                        out[row0 * D + idx] = (typename TL::T)(den == 0.0f ? 0.0f : num / den);
                        continue;
                    }
                    part[h * (D + 4) + d] = num;
                    if (d == 0) {
                        part[h * (D + 4) + D] = M;
                        part[h * (D + 4) + D + 1] = den;
                    }
                }
                return;
            }
            if (r < nh) {
                if (cnt == ns) {
                    const float inv = acc.l == 0.0f ? 0.0f : 1.0f / acc.l;
#pragma unroll
                    for (int e = 0; e < D / 16; e++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            out[(row0 + r) * D + TL::dim(e, gr, i)] = (typename TL::T)(acc.o[e][i] * inv);
                } else {
                    float* p = ws + ((w * 2 + (ci == 0)) * hd.GT + r) * (D + 4);
#pragma unroll
                    for (int e = 0; e < D / 16; e++)
#pragma unroll
                        for (int i = 0; i < 4; i++) p[TL::dim(e, gr, i)] = acc.o[e][i];
                    if (gr == 0) {
                        p[D] = acc.m;
                        p[D + 1] = acc.l;
                    }
                }
            }
        }
        u += cnt;
        ci = 0;
        if (++v == VH && u < u1) {  // the next sequence that has a key: u < u1 <= total, so there is one
            v = 0;
            uint64_t more = __ballot(n > 0) & (sl == 63 ? 0 : ~0ull << (sl + 1));
            while (!more) {
                s0 += 64;
                n = paged_window<TL>(c, lens, s0, lane);
                more = __ballot(n > 0);
            }
            sl = __builtin_ctzll(more);
            ns = (int32_t)lane_of((uint32_t)n, sl);
        }
    }
}

// The wave whose range holds unit u: the last w with floor(total w / W) <= u, that is total w < (u + 1) W.
__device__ __forceinline__ int64_t last_wave(int64_t u, int64_t W, int64_t total)
{
    const uint64_t p = (uint64_t)(u + 1) * (uint64_t)W - 1;
    return (int64_t)((p | (uint64_t)total) >> 32 ? p / (uint64_t)total : (uint32_t)p / (uint32_t)total);
}

// Block (h, s) joins the parts of head h of sequence s: D / 4 lanes a part, 4 dims a lane, each
// group of lanes every S-th part into a running maximum and sums rescaled to it; then the groups of a
// wave by lane shuffles, and the waves through LDS.
// FAST, for caches of codes: exponentials as the hardware has them (of differences of at most 0), and all waves' sums at once,
// with four parts on their way (96 ragged contexts 55.5 -> 54.1 us).  The fp16 and fp32 cache keeps the outputs that it had.
template <typename T, int D, bool FAST>
__global__ __launch_bounds__(1024) void k_attention_paged_merge(int32_t B, T* __restrict__ out, PagedHeads hd, int32_t H,
                                                                const int64_t* __restrict__ before, const float* __restrict__ ws,
                                                                int32_t VH, int32_t waves)
{
    constexpr int L = D / 4, GW = 64 / L;  // lanes a part, parts a wave at a time
    __shared__ f4 so[16][L];
    __shared__ float sm[16], sl[16];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, NW = blockDim.x >> 6, grp = lane / L, d = lane - grp * L;
    const int32_t h = blockIdx.x, s = blockIdx.y, g = h / hd.G, t = (h - g * hd.G) / hd.GT, hr = h - g * hd.G - t * hd.GT;
    const int64_t first = before[s], ns = before[s + 1] - first, total = before[B] * VH;
    T* o4 = out + ((int64_t)s * H + h) * D + 4 * d;
    if (ns == 0) {
        if (wv == 0 && grp == 0)
#pragma unroll
            for (int i = 0; i < 4; i++) o4[i] = (T)0.0f;
        return;
    }
    const int64_t a = first * VH + (g * hd.tiles + t) * ns, b = a + ns - 1;  // first and last unit
    const int64_t W = total < waves ? total : waves;
    // lanes 0 and 1: the waves of units a and b; then where their blocks and the ones after them begin
    const int64_t wl2 = last_wave(lane & 1 ? b : a, W, total), w0 = lane_of64(wl2, 0), w1 = lane_of64(wl2, 1), k0 = w0 / 4, k1 = w1 / 4;
    const uint64_t at = muldiv(total, 4 * ((lane & 1 ? k1 : k0) + (lane >> 1 & 1)), W);
    // its parts: those of the first block's waves (if it is not all in the tile), of the blocks that are, of the last
    // one's waves
    auto inside = [&](int64_t blk, int l) { return 4 * blk + 4 <= W && lane_of64(at, l) >= a && lane_of64(at, l + 2) <= b + 1; };
    const bool in0 = inside(k0, 0), in1 = inside(k1, 1);
    const int64_t lead = in0 ? 0 : (w1 < 4 * k0 + 3 ? w1 : 4 * k0 + 3) - w0 + 1, f0 = k0 + !in0;
    const int64_t full = k1 + in1 > f0 ? k1 + in1 - f0 : 0, parts = lead + full + (k1 == k0 || in1 ? 0 : w1 - 4 * k1 + 1);
    if (parts == 1) return;  // one wave or block had it all
    float M = -INFINITY, den = 0.0f;
    f4 num = {};
    auto join = [&](float m, float l, f4 o) {
        const float mn = fmaxf(M, m), mb = mn == -INFINITY ? 0.0f : mn;
        const float f = FAST ? __builtin_amdgcn_exp2f(M - mb) : exp2f(M - mb), e = FAST ? __builtin_amdgcn_exp2f(m - mb) : exp2f(m - mb);
        num = num * f + o * e;
        den = den * f + l * e;
        M = mn;
    };
    auto part = [&](int64_t i) {
        const int64_t w = i < lead ? w0 + i : i < lead + full ? 4 * (f0 + i - lead) : 4 * k1 + i - lead - full;
        return ws + ((w * 2 + (w == w0)) * hd.GT + hr) * (D + 4);
    };
    if constexpr (FAST) {  // four parts a group on their way at a time, the last ones again where there are fewer
        for (int64_t i0 = wv * GW + (grp < GW ? grp : 0); i0 < parts; i0 += 4 * NW * GW) {
            float m[4], l[4];
            f4 o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t i = i0 + j * NW * GW;
                const float* p = part(i < parts ? i : parts - 1);
                m[j] = p[D];
                l[j] = p[D + 1];
                o[j] = *reinterpret_cast<const f4*>(p + 4 * d);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i0 + j * NW * GW < parts) join(m[j], l[j], o[j]);
        }
    } else if (grp < GW) {
#pragma unroll 4
        for (int64_t i = wv * GW + grp; i < parts; i += NW * GW) {
            const float* p = part(i);
            join(p[D], p[D + 1], *reinterpret_cast<const f4*>(p + 4 * d));
        }
    }
#pragma unroll
    for (int i = 1; i < GW; i++) {  // lanes past the first group's end with sums that nobody reads
        const int from = (lane + i * L) & 63;
        const float m = __shfl(M, from), l = __shfl(den, from);
        const f4 o = {__shfl(num[0], from), __shfl(num[1], from), __shfl(num[2], from), __shfl(num[3], from)};
        if (lane < L) join(m, l, o);
    }
    if (NW > 1) {
        if (lane < L) so[wv][d] = num;
        if (lane == 0) {
            sm[wv] = M;
            sl[wv] = den;
        }
        __syncthreads();
        if (wv > 0) return;
        if (lane < L && !FAST)
            for (int i = 1; i < NW; i++) join(sm[i], sl[i], so[i][d]);
        if (lane < L && FAST) {
            float m[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                m[i] = i < NW ? sm[i] : -INFINITY;
                M = fmaxf(M, m[i]);
            }
            const float mb = M == -INFINITY ? 0.0f : M;
            num = f4{};
            den = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                if (i >= NW) break;
                const float f = __builtin_amdgcn_exp2f(m[i] - mb);
                num += so[i][d] * f;
                den = __builtin_fmaf(sl[i], f, den);
            }
        }
    }
    if (lane < L)
#pragma unroll
        for (int i = 0; i < 4; i++) o4[i] = (T)(den == 0.0f ? 0.0f : num[i] / den);
}

// Floats of the chunk sums ahead of the parts in the workspace.
__attribute__((unused)) static int64_t paged_before_floats(int64_t B) { return (2 * (B + 1) + 3) / 4 * 4; }

}  // namespace

}  // namespace vvh
