// A paged key-value cache held in 8 and 4 bits: the append that rotates and quantises, rows read back as values, and
// attention of one query per sequence over the codes.  A group of G dims of a row is a minimum m, a scale s (fp16 each) and
// codes c that stand for m + s c.  Row r of page p, kv head h is row (p * KVH + h) * P + r of the page arrays: a kv head's
// keys lie together (16 keys of 128 dims in 4 bits are 1 KB), so that attention reads whole lines of them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// Row of the pages that holds position p of sequence s for kv head 0 (head h: h * P further), -1 for none.
__device__ __forceinline__ int64_t paged_q_row(const PagedQArgs& c, int32_t s, int32_t p)
{
    if (s < 0 || s >= c.B || p < 0 || p / c.P >= c.max_pages) return -1;
    const int32_t page = c.table[(int64_t)s * c.max_pages + p / c.P];
    return page < 0 || page >= c.pages ? -1 : (int64_t)page * c.KVH * c.P + p % c.P;
}

// Place of unit u (8 dims) in a key's row of D dims: units of a 32-dim step apart, the steps of one place together.
__device__ __forceinline__ int32_t key_unit(int32_t u, int32_t D) { return (u & 3) * (D / 32) + (u >> 2); }

template <typename T>
struct __attribute__((aligned(16))) Eight {
    T v[8];
};

__device__ __forceinline__ uint32_t scale_pair(float s, float m)
{
    return (uint32_t)__builtin_bit_cast(uint16_t, (f16)s) | (uint32_t)__builtin_bit_cast(uint16_t, (f16)m) << 16;
}
__device__ __forceinline__ float pair_scale(uint32_t x) { return (float)__builtin_bit_cast(h2, x)[0]; }
__device__ __forceinline__ float pair_min(uint32_t x) { return (float)__builtin_bit_cast(h2, x)[1]; }

// Codes of a lane's 8 values, whose group is the `lanes` lanes around it, to `to`; the group's first lane writes {s, m}.
// In 64 bits: a code is a choice between two neighbours, and half of them would be another one where a last bit differs.
__device__ __forceinline__ void quantise8(const float (&x)[8], int bits, int lanes, uint8_t* to, uint32_t* sm, bool first)
{
    float lo = x[0], hi = x[0], z = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        z = __builtin_fmaf(x[i], 0.0f, z);  // NaN for a value that is not finite
    }
    lo = -group_max(-lo, lanes);
    hi = group_max(hi, lanes);
    const bool fine = group_max(z == 0.0f ? 0.0f : 1.0f, lanes) == 0.0f;
    const float top = bits == 8 ? 255.0f : 15.0f;
    const f16 m = (f16)fminf(fmaxf(lo, -65504.0f), 65504.0f);
    const f16 s = (f16)fminf(fmaxf((float)(((double)hi - (double)m) / (double)top), -65504.0f), 65504.0f);
    if (first) *sm = fine ? scale_pair((float)s, (float)m) : 0x7e007e00u;
    uint32_t w[2] = {0, 0};
    if (fine && s != (f16)0.0f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double level = __builtin_rint(((double)x[i] - (double)m) / (double)s);
            const uint32_t c = (uint32_t)fminf(fmaxf((float)level, 0.0f), top);
            if (bits == 8) w[i / 4] |= c << (8 * (i % 4));
            else w[0] |= c << (4 * i);
        }
    }
    if (bits == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(to) = w[0];
}

// A block a token.  Items: 8 dims of a key (its own 8 values and the 8 that the rotation pairs them with), 8 of a value,
// or 8 pairs of a query head.  A group is 4, 8 or 16 lanes in a row of one wave.
template <typename T>
__global__ __launch_bounds__(512) void k_rope_append_paged_q(PagedQArgs c, T* q_out, const T* q, const T* __restrict__ k,
                                                             const T* __restrict__ v, const int32_t* __restrict__ seqs,
                                                             const int32_t* __restrict__ positions, int32_t H,
                                                             const float* __restrict__ rope, int32_t rope_positions)
{
    const int32_t D = c.D, half = D / 2, per = D / 8, kvu = c.KVH * per, items = 2 * kvu + H * (half / 8);
    const int64_t t = blockIdx.x;
    const int32_t s = seqs ? seqs[t] : (int32_t)t, p = positions[t];
    if (rope && p >= rope_positions) return;
    const int64_t row = paged_q_row(c, s, p);
    if (row < 0) return;
    const int lanes = c.group / 8;
    for (int32_t i = threadIdx.x; i < items; i += blockDim.x) {
        if (i < 2 * kvu) {
            const bool key = i < kvu;
            const int32_t h = (key ? i : i - kvu) / per, u = (key ? i : i - kvu) - h * per;
            const T* src = (key ? k : v) + (t * c.KVH + h) * D;
            const Eight<T> a = *reinterpret_cast<const Eight<T>*>(src + 8 * u);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (float)a.v[j];
            if (key && rope) {
                const bool low = 8 * u < half;
                const int32_t d = low ? 8 * u : 8 * u - half;
                const Eight<T> b = *reinterpret_cast<const Eight<T>*>(src + (low ? 8 * u + half : 8 * u - half));
                const f4* cs = reinterpret_cast<const f4*>(rope + ((int64_t)p * half + d) * 2);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const f4 w = cs[j / 2];
                    const double co = w[j % 2 * 2], si = w[j % 2 * 2 + 1];
                    const double o = (double)(float)b.v[j] * (low ? -si : si);  // exact, like the product that it is added to
                    x[j] = (float)__builtin_fma((double)x[j], co, o);
                }
            }
            const int bits = key ? c.kb : c.vb;
            const int64_t r = row + (int64_t)h * c.P;
            uint8_t* to = (key ? c.kp : c.vp) + r * (D * bits / 8) + (key ? key_unit(u, D) : u) * bits;
            uint32_t* sm = (key ? c.ks : c.vs) + r * (D / c.group) + u / lanes;
            quantise8(x, bits, lanes, to, sm, u % lanes == 0);
            continue;
        }
        const int32_t j = i - 2 * kvu, h = j / (half / 8), d = (j - h * (half / 8)) * 8;
        const int64_t at = (t * H + h) * D + d;
        Eight<T> a = *reinterpret_cast<const Eight<T>*>(q + at), b = *reinterpret_cast<const Eight<T>*>(q + at + half);
        const f4* cs = reinterpret_cast<const f4*>(rope + ((int64_t)p * half + d) * 2);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const f4 w = cs[e / 2];
            float r0, r1;
            rope_apply((float)a.v[e], (float)b.v[e], w[e % 2 * 2], w[e % 2 * 2 + 1], r0, r1);
            a.v[e] = (T)r0;
            b.v[e] = (T)r1;
        }
        *reinterpret_cast<Eight<T>*>(q_out + at) = a;
        *reinterpret_cast<Eight<T>*>(q_out + at + half) = b;
    }
}

// A thread 8 dims of a key or a value: a unit of codes, its group's {s, m}, 8 values.  A block a token after another.
template <typename T>
__global__ __launch_bounds__(256) void k_read_paged_q(PagedQArgs c, T* __restrict__ k_out, T* __restrict__ v_out,
                                                      const int32_t* __restrict__ seqs, const int32_t* __restrict__ positions,
                                                      int64_t tokens)
{
    const int32_t D = c.D, per = D / 8, kvu = c.KVH * per, lanes = c.group / 8;
    const int32_t mine = (256 + 2 * kvu - 1) / (2 * kvu);  // tokens of a block
    const int64_t t0 = (int64_t)blockIdx.x * mine;
    const int32_t n = tokens - t0 < mine ? (int32_t)(tokens - t0) : mine;
    for (int32_t i = threadIdx.x; i < n * 2 * kvu; i += 256) {
        const int32_t tt = i / (2 * kvu), j = i - tt * 2 * kvu;
        const bool key = j < kvu;
        T* out = key ? k_out : v_out;
        if (!out) continue;
        const int64_t t = t0 + tt;
        const int64_t row = paged_q_row(c, seqs ? seqs[t] : (int32_t)t, positions[t]);
        if (row < 0) continue;
        const int32_t h = (key ? j : j - kvu) / per, u = (key ? j : j - kvu) - h * per;
        const int bits = key ? c.kb : c.vb;
        const int64_t r = row + (int64_t)h * c.P;
        const uint8_t* at = (key ? c.kp : c.vp) + r * (D * bits / 8) + (key ? key_unit(u, D) : u) * bits;
        const uint32_t sm = (key ? c.ks : c.vs)[r * (D / c.group) + u / lanes];
        const float s = pair_scale(sm), m = pair_min(sm);
        Eight<T> y;
        if (bits == 8) {
            const uint2 w = *reinterpret_cast<const uint2*>(at);
#pragma unroll
            for (int e = 0; e < 8; e++) y.v[e] = (T)__builtin_fmaf(s, (float)((e < 4 ? w.x : w.y) >> (8 * (e % 4)) & 255), m);
        } else {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
            for (int e = 0; e < 8; e++) y.v[e] = (T)__builtin_fmaf(s, (float)(w >> (4 * e) & 15), m);
        }
        *reinterpret_cast<Eight<T>*>(out + (t * c.KVH + h) * D + 8 * u) = y;
    }
}

__device__ __forceinline__ float code_of(const uint8_t* row, int32_t d, int bits, bool key, int32_t D)
{
    if (key) d = key_unit(d / 8, D) * 8 + d % 8;
    return (float)(bits == 8 ? row[d] : row[d / 2] >> (d % 2 * 4) & 15);
}

// softmax(scale q K^T) V of one query head: a block per (head, sequence), its 4 waves each every fourth key, lane l the
// dims l and l + 64; a running maximum m, sum l and numerator o, merged through LDS.
template <typename T>
__global__ __launch_bounds__(256) void k_attention_paged_q(PagedQArgs c, T* __restrict__ out, const T* __restrict__ q,
                                                           const int32_t* __restrict__ lens, int32_t H, float scale)
{
    __shared__ float wm[4], wl[4], wo[4][128];
    const int32_t h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int32_t D = c.D, NG = D / c.group, g = h / (H / c.KVH);
    const int64_t cap = (int64_t)c.max_pages * c.P;
    const int32_t len = lens[s] < 0 ? 0 : lens[s] < cap ? lens[s] : (int32_t)cap;
    const T* qr = q + ((int64_t)s * H + h) * D;
    float x[2], o[2] = {}, m = -INFINITY, l = 0.0f;
    for (int i = 0; i < 2; i++) x[i] = lane + 64 * i < D ? (float)qr[lane + 64 * i] * scale : 0.0f;
    for (int32_t p = w; p < len; p += 4) {
        const int64_t row0 = paged_q_row(c, s, p);
        if (row0 < 0) continue;
        const int64_t row = row0 + (int64_t)g * c.P;
        float d = 0.0f, v[2] = {};
        for (int i = 0; i < 2; i++) {
            const int32_t dim = lane + 64 * i;
            if (dim >= D) continue;
            const uint32_t ks = c.ks[row * NG + dim / c.group], vs = c.vs[row * NG + dim / c.group];
            d += x[i] * __builtin_fmaf(pair_scale(ks), code_of(c.kp + row * (D * c.kb / 8), dim, c.kb, true, D), pair_min(ks));
            v[i] = __builtin_fmaf(pair_scale(vs), code_of(c.vp + row * (D * c.vb / 8), dim, c.vb, false, D), pair_min(vs));
        }
        d = wave_sum_xor(d);
        const float mn = fmaxf(m, d), f = m == -INFINITY ? 0.0f : expf(m - mn), e = expf(d - mn);
        l = l * f + e;
        for (int i = 0; i < 2; i++) o[i] = o[i] * f + e * v[i];
        m = mn;
    }
    if (lane == 0) {
        wm[w] = m;
        wl[w] = l;
    }
    for (int i = 0; i < 2; i++) wo[w][lane + 64 * i] = o[i];
    __syncthreads();
    const float M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    const int32_t d = threadIdx.x;
    if (d >= D) return;
    float num = 0.0f, den = 0.0f;
    for (int i = 0; i < 4; i++) {
        const float f = wm[i] == -INFINITY && wl[i] == 0.0f ? 0.0f : expf(wm[i] - M);
        num = __builtin_fmaf(f, wo[i][d], num);
        den = __builtin_fmaf(f, wl[i], den);
    }
    out[((int64_t)s * H + h) * D + d] = (T)(den == 0.0f ? 0.0f : num / den);
}

// A launch holds fewer than 2^32 threads: at most 2^22 tokens each (of up to 512).
constexpr int64_t kQTokens = int64_t(1) << 22;

}  // namespace

int launch_rope_append_paged_q(const PagedQArgs& c, void* q_out, const void* q, const void* k, const void* v,
                               const int32_t* seqs, const int32_t* positions, int64_t tokens, int64_t H, const float* rope,
                               int64_t rope_positions, int dtype, void* stream)
{
    const int64_t items = 2 * (int64_t)c.KVH * (c.D / 8) + H * (c.D / 16);
    const int64_t threads = std::min<int64_t>((items + 63) / 64 * 64, tokens > 1024 ? 256 : 512);
    auto go = [&](auto kern, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        // without seqs token t is sequence t, of fewer than 2^16: one launch
        for (int64_t t = 0; t < tokens; t += kQTokens) {
            const int64_t qd = t * H * c.D, kd = t * c.KVH * c.D;
            hipLaunchKernelGGL(kern, dim3((unsigned)std::min(tokens - t, kQTokens)), dim3((unsigned)threads), 0,
                               static_cast<hipStream_t>(stream), c, (T*)q_out + (q_out ? qd : 0), (const T*)q + (q ? qd : 0),
                               (const T*)k + kd, (const T*)v + kd, seqs ? seqs + t : nullptr, positions + t, (int32_t)H, rope,
                               (int32_t)rope_positions);
        }
    };
    dtype == VVH_F16 ? go(k_rope_append_paged_q<f16>, (f16*)nullptr) : go(k_rope_append_paged_q<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

int launch_read_paged_q(const PagedQArgs& c, void* k_out, void* v_out, const int32_t* seqs, const int32_t* positions,
                        int64_t tokens, int dtype, void* stream)
{
    const int64_t kvu = (int64_t)c.KVH * (c.D / 8), mine = (256 + 2 * kvu - 1) / (2 * kvu);
    auto go = [&](auto kern, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        for (int64_t t = 0; t < tokens; t += kQTokens) {  // as above
            const int64_t n = std::min(tokens - t, kQTokens), kd = t * c.KVH * c.D;
            hipLaunchKernelGGL(kern, dim3((unsigned)((n + mine - 1) / mine)), dim3(256), 0, static_cast<hipStream_t>(stream), c,
                               (T*)k_out + (k_out ? kd : 0), (T*)v_out + (v_out ? kd : 0), seqs ? seqs + t : nullptr, positions + t, n);
        }
    };
    dtype == VVH_F16 ? go(k_read_paged_q<f16>, (f16*)nullptr) : go(k_read_paged_q<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

int launch_attention_paged_q(const PagedQArgs& c, void* out, const void* q, const int32_t* lens, int64_t H, float scale,
                             int dtype, void* stream)
{
    auto go = [&](auto kern, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        hipLaunchKernelGGL(kern, dim3((unsigned)H, (unsigned)c.B), dim3(256), 0, static_cast<hipStream_t>(stream), c, (T*)out,
                           (const T*)q, lens, (int32_t)H, scale);
    };
    dtype == VVH_F16 ? go(k_attention_paged_q<f16>, (f16*)nullptr) : go(k_attention_paged_q<float>, (float*)nullptr);
    return (int)hipGetLastError();
}

}  // namespace vvh
