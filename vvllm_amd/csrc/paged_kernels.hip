// A key-value cache in pages: the RoPE table, the append of tokens of any
// sequences (rotation of q and k, rows of k and v into their pages) and attention
// of one query per sequence.  Position p of sequence s is row
// table[s * max_pages + p / P] * P + p % P of the pages; a table entry outside
// [0, pages) is no page.
#include <hip/hip_runtime.h>

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

// softmax(scale q K^T) V of one query and head over the pages, any head_dim up to
// 256: a block per (head, sequence), its 4 waves each every fourth position, lane
// l the dims l, l + 64, ...; per position the dot product is summed over the wave
// and joins a running maximum m, sum l and numerator o (o and l rescaled by
// e^(m_old - m)).  The waves' three merge through LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_attention_paged(PagedArgs c, T* __restrict__ out, const T* __restrict__ q,
                                                         const int32_t* __restrict__ lens, int32_t H, float scale)
{
    __shared__ float wm[4], wl[4], wo[4][256];
    const int32_t h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int32_t D = c.D, g = h / (H / c.KVH);
    const int64_t cap = (int64_t)c.max_pages * c.P;
    const int64_t len = lens[s] < cap ? lens[s] : cap;
    const T* qr = q + ((int64_t)s * H + h) * D;
    float x[4], o[4] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = lane + 64 * i < D ? (float)qr[lane + 64 * i] * scale : 0.0f;
    for (int64_t p = w; p < len; p += 4) {
        const int64_t row = paged_row(c, s, (int32_t)p);
        if (row < 0) continue;
        const int64_t at = (row * c.KVH + g) * D + lane;
        float d = 0.0f, vv[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool on = lane + 64 * i < D;
            d = __builtin_fmaf(x[i], on ? (float)((const T*)c.kp)[at + 64 * i] : 0.0f, d);
            vv[i] = on ? (float)((const T*)c.vp)[at + 64 * i] : 0.0f;
        }
        d = wave_sum_xor(d);
        const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.0f : expf(m - mn), e = d == -INFINITY ? 0.0f : expf(d - mn);
        l = __builtin_fmaf(l, f, e);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(o[i], f, e * vv[i]);
        m = mn;
    }
    if (lane == 0) {
        wm[w] = m;
        wl[w] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) wo[w][lane + 64 * i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    float num = 0.0f, den = 0.0f;
    for (int i = 0; i < 4; i++) {
        const float f = wm[i] == -INFINITY ? 0.0f : expf(wm[i] - M);
        num = __builtin_fmaf(f, wo[i][threadIdx.x], num);
        den = __builtin_fmaf(f, wl[i], den);
    }
    if ((int)threadIdx.x < D)
        out[((int64_t)s * H + h) * D + threadIdx.x] = (T)(M == -INFINITY && den == 0.0f ? 0.0f : num / den);
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

int launch_rope_append_paged(const PagedArgs& c, void* q_out, const void* q, const void* k, const void* v,
                             const int32_t* seqs, const int32_t* positions, int64_t tokens, int64_t H,
                             const float* rope, int64_t rope_positions, int dtype, void* stream)
{
    auto go = [&](auto kern, auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(kern, dim3((unsigned)tokens), dim3(256), 0, static_cast<hipStream_t>(stream), c, (T*)q_out,
                           (const T*)q, (const T*)k, (const T*)v, seqs, positions, (int32_t)H, (const float2*)rope,
                           (int32_t)rope_positions);
    };
    dtype == VVH_F16 ? go(k_rope_append_paged<f16>, (f16*)nullptr) : go(k_rope_append_paged<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

int launch_attention_paged(const PagedArgs& c, void* out, const void* q, const int32_t* lens, int64_t H, float scale,
                           int dtype, void* stream)
{
    const dim3 grid((unsigned)H, (unsigned)c.B);
    auto go = [&](auto kern, auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(kern, grid, dim3(256), 0, static_cast<hipStream_t>(stream), c, (T*)out, (const T*)q, lens,
                           (int32_t)H, scale);
    };
    dtype == VVH_F16 ? go(k_attention_paged<f16>, (f16*)nullptr) : go(k_attention_paged<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

}  // namespace vvh
