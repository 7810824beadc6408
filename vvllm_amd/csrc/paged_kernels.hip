// A key-value cache in pages: the RoPE table, the append of tokens of any
// sequences (rotation of q and k, rows of k and v into their pages) and attention
// of one query per sequence.  Position p of sequence s is row
// table[s * max_pages + p / P] * P + p % P of the pages; a table entry outside
// [0, pages) is no page.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

__global__ __launch_bounds__(256) void k_rope_table_theta(float2* __restrict__ out, int64_t n, int32_t half, float theta)
{
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        const int64_t p = e / half, i = e - p * half;
        float c, sn;
        rope_cs(p, i, 2 * (int64_t)half, theta, c, sn);
        out[e] = make_float2(c, sn);
    }
}

// Row of the pages that holds position p of sequence s, -1 for none.
__device__ __forceinline__ int64_t paged_row(const PagedArgs& c, int32_t s, int32_t p)
{
    if (p < 0 || p / c.P >= c.max_pages) return -1;
    const int32_t page = c.table[(int64_t)s * c.max_pages + p / c.P];
    return page < 0 || page >= c.pages ? -1 : (int64_t)page * c.P + p % c.P;
}

// One block per token: its pairs (i, i + D / 2) of every query and key head, then
// its value row.
template <typename T>
__global__ __launch_bounds__(256) void k_rope_append_paged(PagedArgs c, T* q_out, const T* q, const T* __restrict__ k,
                                                           const T* __restrict__ v, const int32_t* __restrict__ seqs,
                                                           const int32_t* __restrict__ positions, int32_t H,
                                                           const float2* __restrict__ rope, int32_t rope_positions)
{
    const int64_t t = blockIdx.x;
    const int32_t s = seqs ? seqs[t] : (int32_t)t, p = positions[t];
    if (s < 0 || s >= c.B || (rope && p >= rope_positions)) return;
    const int64_t row = paged_row(c, s, p);
    if (row < 0) return;
    const int32_t D = c.D, half = D / 2, kv = c.KVH * D;
    T* kr = (T*)c.kp + row * kv;
    T* vr = (T*)c.vp + row * kv;
    const T* kt = k + t * kv;
    const T* vt = v + t * kv;
    if (rope) {
        for (int32_t i = threadIdx.x; i < (H + c.KVH) * half; i += 256) {
            const int32_t h = i / half, d = i - h * half;
            const T* src = h < H ? q + (t * H + h) * D : kt + (h - H) * D;
            T* dst = h < H ? q_out + (t * H + h) * D : kr + (h - H) * D;
            const float2 a = rope[(int64_t)p * half + d];
            float r0, r1;
            rope_apply((float)src[d], (float)src[d + half], a.x, a.y, r0, r1);
            dst[d] = (T)r0;
            dst[d + half] = (T)r1;
        }
    } else {
        for (int32_t i = threadIdx.x; i < kv; i += 256) kr[i] = kt[i];
    }
    for (int32_t i = threadIdx.x; i < kv; i += 256) vr[i] = vt[i];
}

// The same in pieces of 16 bytes: 16 consecutive dims of a head's two halves (8 pairs), or of a value
// row, an item; a block takes a token, and its threads the items.  4001 tokens of 32 query and 8 kv heads of 128 in fp16, 100
// MB: 21.3 us, 4.7 TB/s, a large copy's rate; 8 tokens of 14 and 2 heads of 64: 2.2 us, a launch and its round trips (the
// scalar form above 31 and 7.0).
template <typename T>
struct __attribute__((aligned(16))) Piece {
    T v[8];
};
template <typename T>
__global__ __launch_bounds__(512) void k_rope_append_paged_vec(PagedArgs c, T* q_out, const T* q, const T* __restrict__ k,
                                                                const T* __restrict__ v, const int32_t* __restrict__ seqs,
                                                                const int32_t* __restrict__ positions, int32_t H,
                                                                const float* __restrict__ rope, int32_t rope_positions)
{
    const int32_t D = c.D, half = D / 2, per = half / 8, kv = c.KVH * D;  // items of a head's pairs
    const int32_t heads = H + c.KVH, items = heads * per + kv / 16;
    const int64_t t = blockIdx.x;
    const int32_t s = seqs ? seqs[t] : (int32_t)t, p = positions[t];
    if (s < 0 || s >= c.B || p >= rope_positions) return;
    const int64_t row = paged_row(c, s, p);
    if (row < 0) return;
    for (int32_t i = threadIdx.x; i < items; i += blockDim.x) {
        if (i >= heads * per) {
            const int64_t d = (int64_t)(i - heads * per) * 16;
            const Piece<T> a = *reinterpret_cast<const Piece<T>*>(v + t * kv + d), b = *reinterpret_cast<const Piece<T>*>(v + t * kv + d + 8);
            T* to = (T*)c.vp + row * kv + d;
            *reinterpret_cast<Piece<T>*>(to) = a;
            *reinterpret_cast<Piece<T>*>(to + 8) = b;
            continue;
        }
        const int32_t h = i / per, d = (i - h * per) * 8;
        const T* src = h < H ? q + (t * H + h) * D + d : k + t * kv + (int64_t)(h - H) * D + d;
        T* to = h < H ? q_out + (t * H + h) * D + d : (T*)c.kp + row * kv + (int64_t)(h - H) * D + d;
        Piece<T> a = *reinterpret_cast<const Piece<T>*>(src), b = *reinterpret_cast<const Piece<T>*>(src + half);
        const f4* cs = reinterpret_cast<const f4*>(rope + ((int64_t)p * half + d) * 2);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const f4 x = cs[j];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float r0, r1;
                rope_apply((float)a.v[2 * j + e], (float)b.v[2 * j + e], x[2 * e], x[2 * e + 1], r0, r1);
                a.v[2 * j + e] = (T)r0;
                b.v[2 * j + e] = (T)r1;
            }
        }
        *reinterpret_cast<Piece<T>*>(to) = a;
        *reinterpret_cast<Piece<T>*>(to + half) = b;
    }
}

// softmax(scale q K^T) V of one query and head over the pages, any head_dim up to 256 and any alignment: a block per
// (head, sequence, share of its keys), its 4 waves each every fourth 8 keys, lane l the dims l, l + 64, ... (ND of them).
// The 8 keys' loads are in flight together; a dot product is summed over the wave; they join a running maximum m, sum l
// and numerator o (rescaled by e^(m_old - m)).  The waves' three merge through LDS, the shares' through the
// workspace (a row of D + 2 floats each) in k_attention_paged_any_merge.  8 contexts of 1000 fp16 keys, 16 heads on 8, of 256:
// 66 us (a key at a time, in one block a row: 646), of 80: 25 (385); bound by the 2-byte loads.
template <typename T, int ND>
__global__ __launch_bounds__(256) void k_attention_paged_any(PagedArgs c, T* __restrict__ out, const T* __restrict__ q,
                                                             const int32_t* __restrict__ lens, int32_t H, float scale,
                                                             float* __restrict__ parts)
{
    constexpr int KU = 8;
    __shared__ float wm[4], wl[4], wo[4][64 * ND];
    const int32_t h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6, S = gridDim.z;
    const int32_t D = c.D, g = h / (H / c.KVH);
    const int64_t cap = (int64_t)c.max_pages * c.P;
    const int64_t len = lens[s] < 0 ? 0 : lens[s] < cap ? lens[s] : cap;
    const int32_t p0 = (int32_t)(len * blockIdx.z / S), p1 = (int32_t)(len * (blockIdx.z + 1) / S);
    const T* qr = q + ((int64_t)s * H + h) * D;
    bool on[ND];
    float x[ND], o[ND] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; i++) {
        on[i] = lane + 64 * i < D;
        x[i] = on[i] ? (float)qr[lane + 64 * i] * scale : 0.0f;
    }
    for (int32_t p = p0 + w * KU; p < p1; p += 4 * KU) {
        const int64_t mine = lane < KU && p + lane < p1 ? paged_row(c, s, p + lane) : -1;
        bool live[KU];
        float k[KU][ND], v[KU][ND], d[KU];
#pragma unroll
        for (int j = 0; j < KU; j++) {
            const int32_t row = __builtin_amdgcn_readlane((int)mine, j);
            live[j] = row >= 0;
            const int64_t at = ((int64_t)(row < 0 ? 0 : row) * c.KVH + g) * D + lane;  // no key: row 0, whatever it holds
#pragma unroll
            for (int i = 0; i < ND; i++) {
                k[j][i] = on[i] ? (float)((const T*)c.kp)[at + 64 * i] : 0.0f;
                v[j][i] = on[i] ? (float)((const T*)c.vp)[at + 64 * i] : 0.0f;
            }
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < KU; j++) {
            d[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < ND; i++) d[j] = __builtin_fmaf(x[i], k[j][i], d[j]);
            d[j] = live[j] ? wave_sum_xor(d[j]) : -INFINITY;
            mn = fmaxf(mn, d[j]);
        }
        const float f = m == -INFINITY ? 0.0f : expf(m - mn);
        l *= f;
#pragma unroll
        for (int i = 0; i < ND; i++) o[i] *= f;
#pragma unroll
        for (int j = 0; j < KU; j++) {
            const float e = d[j] == -INFINITY ? 0.0f : expf(d[j] - mn);
            l += e;
#pragma unroll
            for (int i = 0; i < ND; i++) o[i] = __builtin_fmaf(e, live[j] ? v[j][i] : 0.0f, o[i]);
        }
        m = mn;
    }
    if (lane == 0) {
        wm[w] = m;
        wl[w] = l;
    }
#pragma unroll
    for (int i = 0; i < ND; i++) wo[w][lane + 64 * i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    const int32_t d = threadIdx.x;
    if (d >= D) return;
    float num = 0.0f, den = 0.0f;
    for (int i = 0; i < 4; i++) {
        const float f = wm[i] == -INFINITY ? 0.0f : expf(wm[i] - M);
        num = __builtin_fmaf(f, wo[i][d], num);
        den = __builtin_fmaf(f, wl[i], den);
    }
    const int64_t row = (int64_t)s * H + h;
    if (S == 1) {
        out[row * D + d] = (T)(M == -INFINITY && den == 0.0f ? 0.0f : num / den);
        return;
    }
    float* part = parts + (row * S + blockIdx.z) * (D + 2);
    part[d] = num;
    if (d == 0) {
        part[D] = M;
        part[D + 1] = den;
    }
}
// Block r: row r's S shares, 16 / ND groups of 64 ND threads each every 16 / ND-th, then the groups through LDS.
template <typename T, int ND>
__global__ __launch_bounds__(1024) void k_attention_paged_any_merge(T* __restrict__ out, const float* __restrict__ parts, int32_t D, int32_t S)
{
    constexpr int G = 16 / ND;
    __shared__ float wm[G], wl[G], wo[G][64 * ND];
    const int64_t row = blockIdx.x;
    const int32_t d = threadIdx.x % (64 * ND), gr = threadIdx.x / (64 * ND);
    const float* p = parts + row * S * (D + 2);
    float M = -INFINITY, num = 0.0f, den = 0.0f;
#pragma unroll 4
    for (int32_t i = gr; i < S; i += G) {
        const float *part = p + (int64_t)i * (D + 2), m = part[D], l = part[D + 1], o = part[d < D ? d : 0];
        const float mn = fmaxf(M, m), f = M == -INFINITY ? 0.0f : expf(M - mn), e = m == -INFINITY ? 0.0f : expf(m - mn);
        num = __builtin_fmaf(num, f, e * o);
        den = __builtin_fmaf(den, f, e * l);
        M = mn;
    }
    wo[gr][d] = num;
    if (d == 0) {
        wm[gr] = M;
        wl[gr] = den;
    }
    __syncthreads();
    if (gr > 0 || d >= D) return;
    for (int i = 1; i < G; i++) M = fmaxf(M, wm[i]);
    num = den = 0.0f;
    for (int i = 0; i < G; i++) {
        const float f = wm[i] == -INFINITY ? 0.0f : expf(wm[i] - M);
        num = __builtin_fmaf(f, wo[i][d], num);
        den = __builtin_fmaf(f, wl[i], den);
    }
    out[row * D + d] = (T)(M == -INFINITY && den == 0.0f ? 0.0f : num / den);
}

// ---------------------------------------------------------------------------
// The matrix-core form: head_dim 64, 96 or 128, aligned arrays.
//
// A tile is up to 16 query heads of one kv head (GT of its G heads; VH = KVH *
// ceil(G / GT) tiles a sequence).  One wave takes a tile's keys 64 (fp16) or 32
// (fp32) at a time:
//   S^T = K . q^T   A = K rows straight from the pages (lane: key l % 16, 8 or 4 dims of
//                   group l / 16: one 16-byte load), B = the tile's queries in the same
//                   dims.  A lane then has head l % 16's scores of keys 4 (l / 16) + i.
//   softmax         online, in log2 units: maximum (rounded up to an integer: fewer new ones, whose
//                   rescaling is exact) and sum over the lane's scores and the 4 lanes of the head; all of
//                   it in fp32.  fp16: weights are times 2^14, numerators and sums alike, so that those of 2^-38 of the
//                   largest still have a value in fp16 (thousands of small ones make up for a large one).
//   O^T += V^T P^T  B = the lane's own weights (the keys of a product's slots are any as long
//                   as A has the same), A = V^T: fp16 V rows pass through the wave's LDS
//                   region and its transposing read, weights as fp16 pairs high + low (22 bits); fp32 V
//                   rows are loaded in A's layout (lane: 4 or 2 dims of key 4 (l / 16) + i), weights
//                   as they are, on the fp32 matrix instruction.
// A lane finds the row of key c0 + lane in the page table and hands it to the lanes that
// load it.  A key past the end or on no page loads row 0 instead; its score becomes
// -infinity and its value 0, whatever that row holds.
//
// Infinite values: inf w is the infinity for a weight above 0 (fp32), but the low part of an fp16 pair is 0 or below it
// and makes a NaN of it.  A wave whose fp16 sums are not finite therefore takes its chunks once more (INF), the infinities
// apart from the pairs, against 1 where the weight is above 0; all others pay one test of their sums at the end (16 contexts of
// 4000 keys, 12 heads on 2 of 96, 16.7 -> 16.9 us; 96 contexts from 1 to 8192 keys 84.5 -> 85.2).  The second pass costs what
// the first does (one of 30000 keys 29 -> 47).  A head whose weights' sum is not finite gives NaN without it.
// ---------------------------------------------------------------------------
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ h4 lds_tr16(const f16* p)
{
    typedef short s4v __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(p)));
}

template <typename T>
struct PagedTile;

// CH: keys at a time
template <>
struct PagedTile<f16> {
    template <int D>
    static constexpr int CH = D == 64 ? 64 : 32;
    template <int D>
    struct Q {
        h8 b[D / 32];
    };
    template <int D>
    static constexpr int lds = CH<D> * (D + 4);  // elements of a wave's V region
};
template <>
struct PagedTile<float> {
    template <int D>
    static constexpr int CH = D == 128 ? 16 : 32;
    template <int D>
    struct Q {
        f4 b[D / 16];
    };
    template <int D>
    static constexpr int lds = 0;
};

template <int D>
__device__ __forceinline__ void paged_load_q(const f16* q, int heads, int lane, PagedTile<f16>::Q<D>& x)
{
#pragma unroll
    for (int s = 0; s < D / 32; s++)
        x.b[s] = (lane & 15) < heads ? *reinterpret_cast<const h8*>(q + (lane & 15) * D + 32 * s + 8 * (lane >> 4)) : h8{};
}
template <int D>
__device__ __forceinline__ void paged_load_q(const float* q, int heads, int lane, PagedTile<float>::Q<D>& x)
{
#pragma unroll
    for (int s = 0; s < D / 16; s++)
        x.b[s] = (lane & 15) < heads ? *reinterpret_cast<const f4*>(q + (lane & 15) * D + 16 * s + 4 * (lane >> 4)) : f4{};
}

// Head (lane % 16)'s running maximum, sum and output fragments: o[e][i] is dim
// paged_dim(e, lane / 16, i).
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
template <typename T, int D>
__device__ __forceinline__ constexpr int paged_dim(int e, int gr, int i)
{
    if (sizeof(T) == 2) return 16 * e + 4 * gr + i;
    constexpr int VW = D % 64 == 0 ? 4 : 2;  // dims of a lane's V load
    return 16 * VW * (e / VW) + VW * (4 * gr + i) + e % VW;
}

// The chunks c0, c0 + cstep, ... below ke of sequence s.  kh, vh: the kv head's column
// in the pages; vw: the wave's LDS region (fp16).  BIG: the pages of K or V pass 4 GB, the reach of a
// buffer load's 32-bit offset, and take 64-bit addresses (16 clocks of multiplication a load).  INF (fp16): infinite values
// apart.
template <typename T, int D, bool BIG, bool INF>
__device__ __forceinline__ void paged_chunks(const PagedArgs& c, const T* kh, const T* vh, int32_t s,
                                             const typename PagedTile<T>::template Q<D>& q, int32_t c0, int32_t cstep,
                                             int32_t ke, float scale_log2, f16* vw, int lane, PagedAcc<D>& acc)
{
    constexpr int CH = PagedTile<T>::template CH<D>, NT = CH / 16;
    constexpr bool H16 = sizeof(T) == 2;
    constexpr int DS = H16 ? D / 32 : D / 16, DE = D / 16, VP = D + 4;
    constexpr int VW = D % 64 == 0 ? 4 : 2, VJ = D / (16 * VW);
    typedef float vf __attribute__((ext_vector_type(VW)));
    const int r = lane & 15, gr = lane >> 4;
    const int64_t kvs = (int64_t)c.KVH * D;
    const int32_t* table = c.table + (int64_t)s * c.max_pages;
    const uint64_t pool = (uint64_t)c.pages * c.P * kvs;  // values; a resource ends with the pages
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(kh), 0, BIG ? 0 : (int)(uint32_t)((pool - (uint64_t)(kh - (const T*)c.kp)) * sizeof(T)), 0x00020000);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(vh), 0, BIG ? 0 : (int)(uint32_t)((pool - (uint64_t)(vh - (const T*)c.vp)) * sizeof(T)), 0x00020000);
    const uint32_t stride = (uint32_t)kvs * (uint32_t)sizeof(T);
    // The page of key at + lane and its row there, looked up a chunk ahead (the first one without waiting for the
    // length) and turned into a row of the pages (-1: no key, or no page) only when it is used, so that nothing
    // waits for it.
    const uint32_t cap = (uint32_t)c.max_pages * (uint32_t)c.P;
    struct Spot {
        int32_t page, in;
    };
    auto look = [&](int32_t at) {
        const uint32_t want = (uint32_t)(at + lane), key = want < cap ? want : cap - 1, pg = key / (uint32_t)c.P;
        return Spot{table[pg], (int32_t)(key - pg * (uint32_t)c.P)};
    };
    Spot spot = look(c0);
    for (; c0 < ke; c0 += cstep) {
        const int32_t row = lane < CH && c0 + lane < ke && spot.page >= 0 && spot.page < c.pages ? spot.page * c.P + spot.in : -1;
        const uint64_t live = __ballot(row >= 0);
        const bool all = live == ~0ull >> (64 - CH);
        // every lane's row (its byte offset) to the lanes that load it, all at once
        const uint32_t at = row < 0 ? 0u : BIG ? (uint32_t)row : (uint32_t)row * stride;
        constexpr int NVR = H16 ? CH * D / 512 : NT * 4;
        uint32_t ak[NT], av[NVR];
#pragma unroll
        for (int t = 0; t < NT; t++) ak[t] = (uint32_t)__shfl((int)at, 16 * t + r);
#pragma unroll
        for (int i = 0; i < NVR; i++) av[i] = (uint32_t)__shfl((int)at, H16 ? (i * 64 + lane) / (D / 8) : 16 * (i / 4) + 4 * gr + i % 4);
        __builtin_amdgcn_sched_barrier(0);
        // 16 bytes (or 8) at byte `in` of a row
        auto load16 = [&](const __amdgpu_buffer_rsrc_t& res, const T* col, uint32_t a, int in) {
            if constexpr (BIG) return *reinterpret_cast<const u4*>(reinterpret_cast<const char*>(col + (int64_t)a * kvs) + in);
            else return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(res, a + in, 0, 0));
        };
        f4 sc[NT];
        typename std::conditional<H16, h8, f4>::type ka[NT][DS];
        h8 vr[H16 ? CH * D / 512 : 1];
        vf vv[H16 ? 1 : NT][H16 ? 1 : 4][VJ];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int x = 0; x < DS; x++)
                ka[t][x] = __builtin_bit_cast(typename std::conditional<H16, h8, f4>::type, load16(rk, kh, ak[t], 64 * x + 16 * gr));
        if constexpr (H16) {
#pragma unroll
            for (int i = 0; i < CH * D / 512; i++)
                vr[i] = __builtin_bit_cast(h8, load16(rv, vh, av[i], (i * 64 + lane) % (D / 8) * 16));
        } else {
#pragma unroll
            for (int i = 0; i < NT * 4; i++)
#pragma unroll
                for (int x = 0; x < VJ; x++) {
                    const int in = (16 * VW * x + VW * r) * 4;
                    if constexpr (VW == 4) {
                        vv[i / 4][i % 4][x] = __builtin_bit_cast(vf, load16(rv, vh, av[i], in));
                    } else if constexpr (BIG) {
                        vv[i / 4][i % 4][x] = *reinterpret_cast<const vf*>(vh + (int64_t)av[i] * kvs + in / 4);
                    } else {
                        const uint32_t off = av[i] + in;
                        vv[i / 4][i % 4][x] = __builtin_bit_cast(vf, __builtin_amdgcn_raw_buffer_load_b64(rv, off, 0, 0));
                    }
                }
        }
        spot = look(c0 + cstep);
        // all of the chunk's loads before its first product: fp32 heads of 96 30.0 -> 28.0 us (4 contexts of 8000 keys); the others are
        // as fast either way, or slower for it (fp16 heads of 64, 1000 keys, 8.3 -> 8.9)
        if constexpr (!H16 && D == 96) __builtin_amdgcn_sched_barrier(0);
        // the page lookup on its way first and one wait for all of K, while V and the lookup stay in flight: fp16 heads of 64, 1000
        // keys, 8.3 us, left to the scheduler 8.8
        if constexpr (H16 && !INF && D == 64) {
            __builtin_amdgcn_sched_barrier(0);
            wait_loads<CH * D / 512 + 1>();
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            sc[t] = f4{};
#pragma unroll
            for (int x = 0; x < DS; x++) {
                if constexpr (H16) {
                    sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][x], q.b[x], sc[t], 0, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[t][x][j], q.b[x][j], sc[t], 0, 0, 0);
                }
            }
        }
        float cm = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float x = sc[t][i] * scale_log2;
                if (!all && !(live >> (16 * t + 4 * gr + i) & 1)) x = -INFINITY;
                sc[t][i] = x;
                cm = fmaxf(cm, x);
            }
        cm = max_x32(max_x16(cm));
        if (__any(cm > acc.m)) {  // a new maximum for some head
            const float mn = __builtin_ceilf(fmaxf(acc.m, cm)), f = acc.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(acc.m - mn);
            acc.l *= f;
            acc.m = mn;
#pragma unroll
            for (int e = 0; e < DE; e++) acc.o[e] *= f;
        }
        const float mb = acc.m == -INFINITY ? 0.0f : acc.m - (H16 ? 14.0f : 0.0f);  // no key yet: every weight below is 0
        float ps = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sc[t][i] = __builtin_amdgcn_exp2f(sc[t][i] - mb);
                ps += sc[t][i];
            }
        acc.l += sum_x32(sum_x16(ps));
        if constexpr (H16) {
            if (!all) {
#pragma unroll
                for (int i = 0; i < CH * D / 512; i++)
                    if (!(live >> ((i * 64 + lane) / (D / 8)) & 1)) vr[i] = h8{};
            }
            // the reads below see these rows, and the next chunk's writes come after them
            wave_lds_order();
#pragma unroll
            for (int i = 0; i < CH * D / 512; i++) {
                const int p = i * 64 + lane, j = p / (D / 8), col = p % (D / 8) * 8;
                *reinterpret_cast<h4*>(vw + j * VP + col) = h4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]};
                *reinterpret_cast<h4*>(vw + j * VP + col + 4) = h4{vr[i][4], vr[i][5], vr[i][6], vr[i][7]};
            }
            wave_lds_order();
#pragma unroll
            for (int u = 0; u < NT / 2; u++) {
                h8 hi, lo, on;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float w = sc[2 * u + j / 4][j % 4];
                    hi[j] = (f16)w;
                    lo[j] = (f16)(w - (float)hi[j]);
                    if constexpr (INF) on[j] = (f16)(w > 0.0f ? 1.0f : 0.0f);
                }
                // lane (r, gr): V[32 u + 4 gr + j][16 e + r] and the same 16 keys on, j < 4: in each
                // group of 16 lanes the transposing read gives lane i element i % 4 of lane 4 j + i / 4's
                // piece, so lane s points at dims 16 e + 4 (s % 4) of key 4 gr + s / 4
#pragma unroll
                for (int e = 0; e < DE; e++) {
                    const f16* src = vw + (32 * u + 4 * gr + (r >> 2)) * VP + 16 * e + 4 * (r & 3);
                    const h4 a = lds_tr16(src), b = lds_tr16(src + 16 * VP);
                    h8 va = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                    if constexpr (INF) {
                        h8 vi;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const bool is = __builtin_fabsf((float)va[j]) == INFINITY;
                            vi[j] = is ? va[j] : (f16)0.0f;
                            va[j] = is ? (f16)0.0f : va[j];
                        }
                        acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vi, on, acc.o[e], 0, 0, 0);
                    }
                    acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, hi, acc.o[e], 0, 0, 0);
                    acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, lo, acc.o[e], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (!all && !(live >> (16 * t + 4 * gr + i) & 1)) {
#pragma unroll
                        for (int x = 0; x < VJ; x++) vv[t][i][x] = vf{};
                    }
#pragma unroll
                    for (int e = 0; e < DE; e++)
                        acc.o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[t][i][e / VW][e % VW], sc[t][i], acc.o[e], 0, 0, 0);
                }
        }
    }
}

// The chunks, and once more where a sum of the wave is not finite although its weights' sum is
template <typename T, int D, bool BIG>
__device__ __forceinline__ void paged_tile(const PagedArgs& c, const T* kh, const T* vh, int32_t s,
                                           const typename PagedTile<T>::template Q<D>& q, int32_t c0, int32_t cstep,
                                           int32_t ke, float scale_log2, f16* vw, int lane, PagedAcc<D>& acc)
{
    acc.clear();
    paged_chunks<T, D, BIG, false>(c, kh, vh, s, q, c0, cstep, ke, scale_log2, vw, lane, acc);
    if constexpr (sizeof(T) == 2) {
        f4 z = {};  // 0, or NaN; four chains
#pragma unroll
        for (int e = 0; e < D / 16; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) z[i] = __builtin_fmaf(acc.o[e][i], 0.0f, z[i]);
        if (__builtin_expect(!__any((z[0] + z[1]) + (z[2] + z[3]) != 0.0f && acc.l - acc.l == 0.0f), 1)) return;
        // nothing of this pass is worked out ahead of the first one (16 contexts of 4000 keys of 96 17.1 -> 16.9 us)
        PagedArgs c2 = c;
        asm volatile("" : "+s"(c2.P), "+s"(c2.KVH), "+s"(c2.max_pages), "+s"(c2.pages), "+s"(c2.table));
        const int lane2 = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));
        acc.clear();
        paged_chunks<T, D, BIG, true>(c2, kh, vh, s, q, c0, cstep, ke, scale_log2, vw, lane2, acc);
    }
}

// Sequence s's length, as the kernels take it
__device__ __forceinline__ int32_t paged_len(const PagedArgs& c, const int32_t* lens, int32_t s)
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

// One tile of one sequence by one block, its NW waves each every NW-th chunk, merged
// through LDS: short contexts, in one launch.  4 chats of up to 512 fp16 keys, 14 heads on 2 of 64: 5.8 us, of which a launch
// and the round trips for lengths and pages, rows, and the merge; 1.1 MB is not what bounds it.
template <typename T, int D, int NW, bool BIG>
__global__ __launch_bounds__(64 * NW, 2) void k_attention_paged_one(PagedArgs c, T* __restrict__ out, const T* __restrict__ q,
                                                                 const int32_t* __restrict__ lens, PagedHeads hd, int32_t H,
                                                                 float scale_log2)
{
    constexpr int CH = PagedTile<T>::template CH<D>, OP = D + 4;
    constexpr int VB = PagedTile<T>::template lds<D> * 2, OB = 16 * OP * 4;  // bytes a wave
    __shared__ __align__(16) char smem[NW * (VB > OB ? VB : OB)];
    __shared__ float wm[NW][16], wl[NW][16];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, gr = lane >> 4;
    const int32_t s = blockIdx.y, len = paged_len(c, lens, s);
    int32_t g, h0, n;
    hd.at(blockIdx.x, g, h0, n);
    const int64_t row0 = (int64_t)s * H + h0;
    typename PagedTile<T>::template Q<D> x;
    paged_load_q<D>(q + row0 * D, n, lane, x);
    PagedAcc<D> acc;
    paged_tile<T, D, BIG>(c, (const T*)c.kp + g * D, (const T*)c.vp + g * D, s, x, w * CH, NW * CH, len, scale_log2,
                          reinterpret_cast<f16*>(smem + w * VB), lane, acc);
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);
    if (gr == 0) {
        wm[w][r] = acc.m;
        wl[w][r] = acc.l;
    }
#pragma unroll
    for (int e = 0; e < D / 16; e++)
#pragma unroll
        for (int i = 0; i < 4; i++) os[(w * 16 + r) * OP + paged_dim<T, D>(e, gr, i)] = acc.o[e][i];
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
        out[row0 * D + idx] = (T)(den == 0.0f ? 0.0f : num / den);
    }
}

// Chunks of the 64 sequences from s0 on, one a lane, and their sums up to each lane.
__device__ __forceinline__ int32_t paged_window(const PagedArgs& c, const int32_t* lens, int32_t s0, int lane, int ch)
{
    return s0 + lane < c.B ? (paged_len(c, lens, s0 + lane) + ch - 1) / ch : 0;
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
// With the merge: 96 contexts from 1 to 8192 fp16 keys, 32 heads on 8 of 128, 373 MB in 85 us, 4.4 TB/s; 32 of 4096, 8 heads on
// 8, 537 MB in 101 us, 5.3 TB/s; 3 of up to 30001 fp32 keys, 12 heads on 2, 153 MB in 41 us, 3.7 TB/s.  Bound by HBM; about 7
// us of the first and last are the merge's launch and round trips.
template <typename T, int D, bool BIG>
__global__ __launch_bounds__(256, 2) void k_attention_paged_split(PagedArgs c, T* __restrict__ out, const T* __restrict__ q,
                                                               const int32_t* __restrict__ lens, PagedHeads hd, int32_t H,
                                                               float scale_log2, int64_t* __restrict__ before_out, float* __restrict__ ws,
                                                                  int32_t VH)
{
    constexpr int CH = PagedTile<T>::template CH<D>;
    constexpr int VB = PagedTile<T>::template lds<D> * 2, OP = D + 4, OB = 16 * OP * 4;  // bytes a wave
    __shared__ __align__(16) char smem[4 * (VB > OB ? VB : OB)];
    __shared__ float wm[4][16], wl[4][16];
    const int lane = threadIdx.x & 63, r = lane & 15, gr = lane >> 4;
    const int wb = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = (int64_t)blockIdx.x * 4 + wb;
    // the sums of the chunks before each sequence, and of all: the first wave keeps them for the merge
    int64_t total = 0;
    for (int32_t s0 = 0; s0 < c.B; s0 += 64) {
        const uint32_t upto = wave_scan((uint32_t)paged_window(c, lens, s0, lane, CH));  // at most 64 * 2^25
        if (w == 0 && s0 + lane < c.B) before_out[s0 + lane + 1] = total + upto;
        total += lane_of(upto, 63);
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
    int32_t s0 = 0, n = paged_window(c, lens, 0, lane, CH);
    int64_t before = 0;
    uint32_t upto = wave_scan((uint32_t)n);
    while ((before + lane_of(upto, 63)) * VH <= u0) {
        before += lane_of(upto, 63);
        s0 += 64;
        n = paged_window(c, lens, s0, lane, CH);
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
        typename PagedTile<T>::template Q<D> x;
        paged_load_q<D>(q + row0 * D, nh, lane, x);
        PagedAcc<D> acc;
        const int32_t len = __builtin_amdgcn_readfirstlane(paged_len(c, lens, s));
        const int64_t end = (int64_t)(ci + cnt) * CH;
        paged_tile<T, D, BIG>(c, (const T*)c.kp + g * D, (const T*)c.vp + g * D, s, x, ci * CH, CH,
                              end < len ? (int32_t)end : len, scale_log2, reinterpret_cast<f16*>(smem + wb * VB), lane, acc);
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
                for (int i = 0; i < 4; i++) os[(wb * 16 + r) * OP + paged_dim<T, D>(e, gr, i)] = acc.o[e][i];
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
                    out[row0 * D + idx] = (T)(den == 0.0f ? 0.0f : num / den);
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
                        out[(row0 + r) * D + paged_dim<T, D>(e, gr, i)] = (T)(acc.o[e][i] * inv);
            } else {
                float* p = ws + ((w * 2 + (ci == 0)) * hd.GT + r) * (D + 4);
#pragma unroll
                for (int e = 0; e < D / 16; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) p[paged_dim<T, D>(e, gr, i)] = acc.o[e][i];
                if (gr == 0) {
                    p[D] = acc.m;
                    p[D + 1] = acc.l;
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
                n = paged_window(c, lens, s0, lane, CH);
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
template <typename T, int D>
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
        const float f = exp2f(M - mb), e = exp2f(m - mb);
        num = num * f + o * e;
        den = den * f + l * e;
        M = mn;
    };
    if (grp < GW) {
#pragma unroll 4
        for (int64_t i = wv * GW + grp; i < parts; i += NW * GW) {
            const int64_t w = i < lead ? w0 + i : i < lead + full ? 4 * (f0 + i - lead) : 4 * k1 + i - lead - full;
            const float* p = ws + ((w * 2 + (w == w0)) * hd.GT + hr) * (D + 4);
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
        if (lane < L)
            for (int i = 1; i < NW; i++) join(sm[i], sl[i], so[i][d]);
    }
    if (lane < L)
#pragma unroll
        for (int i = 0; i < 4; i++) o4[i] = (T)(den == 0.0f ? 0.0f : num[i] / den);
}

}  // namespace

int launch_rope_table_theta(float* out, int64_t positions, int64_t D, float theta, void* stream)
{
    const int64_t n = positions * (D / 2);
    const unsigned blocks = (unsigned)((n + 255) / 256 < 65536 ? (n + 255) / 256 : 65536);
    hipLaunchKernelGGL(k_rope_table_theta, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                       reinterpret_cast<float2*>(out), n, (int32_t)(D / 2), theta);
    return (int)hipGetLastError();
}

// A launch holds fewer than 2^32 threads: at most 2^22 tokens each (of up to 512).
constexpr int64_t kAppendTokens = int64_t(1) << 22;

static int launch_append_part(const PagedArgs& c, void* q_out, const void* q, const void* k, const void* v,
                              const int32_t* seqs, const int32_t* positions, int64_t tokens, int64_t H,
                              const float* rope, int64_t rope_positions, int dtype, void* stream)
{
    const uintptr_t all = (uintptr_t)q_out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)c.kp | (uintptr_t)c.vp | (uintptr_t)rope;
    if (rope && c.D % 16 == 0 && all % 16 == 0) {
        const int64_t items = (H + c.KVH) * (c.D / 16) + (int64_t)c.KVH * c.D / 16;
        // many tokens fill the device with 256 threads each (4001 tokens of 32 / 8 heads of 128 23.1 -> 21.7 us), few
        // take more (256 tokens 3.65 -> 3.34)
        const int64_t threads = std::min<int64_t>((items + 63) / 64 * 64, tokens > 1024 ? 256 : 512);
        auto go = [&](auto kern, auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            hipLaunchKernelGGL(kern, dim3((unsigned)tokens), dim3((unsigned)threads), 0, static_cast<hipStream_t>(stream), c, (T*)q_out,
                               (const T*)q, (const T*)k, (const T*)v, seqs, positions, (int32_t)H, rope,
                               (int32_t)rope_positions);
        };
        dtype == VVH_F16 ? go(k_rope_append_paged_vec<f16>, (f16*)nullptr) : go(k_rope_append_paged_vec<float>, (float*)nullptr);
        return (int)hipGetLastError();
    }
    auto go = [&](auto kern, auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(kern, dim3((unsigned)tokens), dim3(256), 0, static_cast<hipStream_t>(stream), c, (T*)q_out,
                           (const T*)q, (const T*)k, (const T*)v, seqs, positions, (int32_t)H, (const float2*)rope,
                           (int32_t)rope_positions);
    };
    dtype == VVH_F16 ? go(k_rope_append_paged<f16>, (f16*)nullptr) : go(k_rope_append_paged<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

int launch_rope_append_paged(const PagedArgs& c, void* q_out, const void* q, const void* k, const void* v,
                             const int32_t* seqs, const int32_t* positions, int64_t tokens, int64_t H,
                             const float* rope, int64_t rope_positions, int dtype, void* stream)
{
    // without seqs token t is sequence t, of fewer than 2^16: one launch
    const int64_t e = dtype == VVH_F16 ? 2 : 4, qb = H * c.D * e, kvb = (int64_t)c.KVH * c.D * e;
    for (int64_t t = 0; t < tokens; t += kAppendTokens) {
        auto at = [&](const void* p, int64_t row) { return p ? (const char*)p + t * row : nullptr; };
        const int st = launch_append_part(c, (void*)at(q_out, qb), at(q, qb), at(k, kvb), at(v, kvb), seqs ? seqs + t : nullptr,
                                          positions + t, std::min(tokens - t, kAppendTokens), H, rope, rope_positions, dtype, stream);
        if (st != 0) return st;
    }
    return 0;
}


// A block takes up to two chunks a wave of a context by itself (400 fp16 keys of 128, 8 contexts, 8.9 us, split 11.2), more
// are split (three a wave: 400 fp32 keys of 128 13.6 -> 11.4; four: 32 contexts of up to 1000 fp16 keys 15.5 -> 11.9).
constexpr int64_t kPagedOneChunks = 16;

// Floats of the chunk sums ahead of the parts in the workspace.
static int64_t paged_before_floats(int64_t B) { return (2 * (B + 1) + 3) / 4 * 4; }

static bool attention_paged_tiled(const PagedArgs& c, const void* q, int dtype)
{
    const uintptr_t all = (uintptr_t)c.kp | (uintptr_t)c.vp | (uintptr_t)q;
    return (c.D == 64 || c.D == 96 || c.D == 128) && all % 16 == 0 && (dtype == VVH_F16 || dtype == VVH_F32);
}

AttnPagedPlan attention_paged_plan(const PagedArgs& c, const void* q, int64_t max_len, int64_t H, int dtype,
                                   int64_t cus)
{
    AttnPagedPlan p{};
    const int64_t G = H / c.KVH;
    p.tiled = attention_paged_tiled(c, q, dtype);
    p.tiles = (G + 15) / 16;
    p.GT = (G + p.tiles - 1) / p.tiles;
    const int64_t cap = (int64_t)c.max_pages * c.P;
    const int64_t len = max_len > 0 && max_len < cap ? max_len : cap;
    if (!p.tiled) {  // shares of at least 64 keys, to about 8 blocks a CU (8 contexts of 1000 keys of 80 24.8 us, to 4 a CU 34.3, to 2 57)
        p.blocks = std::max<int64_t>(1, std::min<int64_t>({(len + 63) / 64, (8 * cus + c.B * H - 1) / (c.B * H), 256}));
        p.ws_floats = p.blocks > 1 ? c.B * H * p.blocks * (c.D + 2) : 0;
        return p;
    }
    const int64_t ch = dtype == VVH_F16 ? (c.D == 64 ? PagedTile<f16>::CH<64> : PagedTile<f16>::CH<128>)
                                        : (c.D == 128 ? PagedTile<float>::CH<128> : PagedTile<float>::CH<64>);
    const int64_t chunks = (len + ch - 1) / ch;
    p.waves = chunks > 4 ? 8 : 4;
    if (chunks > kPagedOneChunks) {
        // a chunk a wave at least (one context of 3000 keys, fp32 heads of 128, a wave every 4 chunks 17.9 us, every 2 14.9,
        // every one 12.4), and two blocks a CU; fp16 of one sequence one, whose waves then have longer runs (30000 keys
        // 18.9 -> 17.0 us, but 8 ragged contexts of up to 8000 keys 12.4 -> 13.5, 96 84.5 -> 92)
        p.blocks = std::min<int64_t>((chunks * c.B * c.KVH * p.tiles + 3) / 4, (dtype == VVH_F16 && c.B == 1 ? 1 : 2) * cus);
    }
    if (p.blocks > 0) p.ws_floats = paged_before_floats(c.B) + p.blocks * 4 * 2 * p.GT * (c.D + 4);
    return p;
}

template <typename T, int D, bool BIG>
static void paged_go(const AttnPagedPlan& p, const PagedArgs& c, T* out, const T* q, const int32_t* lens, int64_t H,
                     float scale_log2, float* ws, hipStream_t s)
{
    const PagedHeads hd{(int32_t)(H / c.KVH), (int32_t)p.GT, (int32_t)p.tiles};
    const int32_t VH = (int32_t)(c.KVH * p.tiles);
    if (p.blocks == 0) {
        auto one = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3((unsigned)VH, (unsigned)c.B), dim3((unsigned)(64 * p.waves)), 0, s, c, out, q, lens, hd,
                               (int32_t)H, scale_log2);
        };
        p.waves == 8 ? one(k_attention_paged_one<T, D, 8, BIG>) : one(k_attention_paged_one<T, D, 4, BIG>);
        return;
    }
    int64_t* before = reinterpret_cast<int64_t*>(ws);
    float* parts = ws + paged_before_floats(c.B);
    hipLaunchKernelGGL((k_attention_paged_split<T, D, BIG>), dim3((unsigned)p.blocks), dim3(256), 0, s, c, out, q, lens, hd,
                       (int32_t)H, scale_log2, before, parts, VH);
    // waves of a merge block: about 4 parts a group of lanes if the sequences are alike
    const int64_t W = p.blocks * 4;
    int64_t nw = 1;
    while (nw < 16 && nw * (256 / D) * 4 < p.blocks / ((int64_t)VH * c.B)) nw *= 2;
    hipLaunchKernelGGL((k_attention_paged_merge<T, D>), dim3((unsigned)H, (unsigned)c.B), dim3((unsigned)(64 * nw)), 0, s,
                       (int32_t)c.B, out, hd, (int32_t)H, before, parts, VH, (int32_t)W);
}

int launch_attention_paged(const AttnPagedPlan& p, const PagedArgs& c, void* out, const void* q, const int32_t* lens, int64_t H,
                           float scale, float* ws, int dtype, void* stream)
{
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (p.tiled) {
            const float sl = (float)((double)scale * 1.4426950408889634);  // scores in log2 units
            auto run = [&](auto d) {
                constexpr int D = decltype(d)::value;
                const bool big = (uint64_t)c.pages * c.P * c.KVH * D * sizeof(T) > UINT32_MAX;
                if (big) paged_go<T, D, true>(p, c, (T*)out, (const T*)q, lens, H, sl, ws, st);
                else paged_go<T, D, false>(p, c, (T*)out, (const T*)q, lens, H, sl, ws, st);
            };
            c.D == 64 ? run(std::integral_constant<int, 64>{}) : c.D == 96 ? run(std::integral_constant<int, 96>{}) : run(std::integral_constant<int, 128>{});
        } else {
            auto any = [&](auto nd) {
                constexpr int ND = decltype(nd)::value;
                hipLaunchKernelGGL((k_attention_paged_any<T, ND>), dim3((unsigned)H, (unsigned)c.B, (unsigned)p.blocks), dim3(256), 0, st, c,
                                   (T*)out, (const T*)q, lens, (int32_t)H, scale, ws);
                if (p.blocks > 1)
                    hipLaunchKernelGGL((k_attention_paged_any_merge<T, ND>), dim3((unsigned)(c.B * H)), dim3(1024), 0, st, (T*)out,
                                       (const float*)ws, c.D, (int32_t)p.blocks);
            };
            c.D <= 64 ? any(std::integral_constant<int, 1>{})
            : c.D <= 128 ? any(std::integral_constant<int, 2>{}) : any(std::integral_constant<int, 4>{});
        }
    };
    dtype == VVH_F16 ? go((f16*)nullptr) : go((float*)nullptr);
    return (int)hipGetLastError();
}

}  // namespace vvh
