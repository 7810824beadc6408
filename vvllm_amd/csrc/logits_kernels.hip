// The rules between a row of logits and its sampler: penalties of tokens that were
// there before, biases, and a mask of allowed tokens.
#include <hip/hip_runtime.h>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// N values in one access (two for 8 floats), of any alignment (a row of an odd vocabulary, a history)
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Some {
    T v[N];
};
// Block (x, r): the `span` logits of row r from x * span on, 8 a thread.  It counts the row's tokens that fall into its
// span (bit 31: seen at all; below it the times among those after the prompt; sums of integers, so in any
// order) and finds each biased token's last entry, then takes its logits through the rules.
// cnt: a word of LDS a logit, entry: as many if there are biases.  64 rows of 151936 fp16 logits with masks, histories of up
// to 4000 tokens and 300 biases each, 41 MB: 15.9 us, 2.6 TB/s, of which 8 us is what the logits and masks alone take (HBM) and 4
// each the histories and the biases (LDS and the barriers between them); one fp32 row 3.9 us, a launch and two round trips.
template <typename T>
__global__ __launch_bounds__(1024) void k_logits_rules(T* out, const T* logits, vvh_logits_spec a, int32_t n)
{
    const int32_t threads = blockDim.x, span = 8 * threads;
    extern __shared__ __align__(16) uint32_t cnt[];
    int32_t* entry = reinterpret_cast<int32_t*>(cnt + span);
    const int32_t r = blockIdx.y, i0 = blockIdx.x * span, tid = threadIdx.x;
    const int32_t len = n - i0 < span ? n - i0 : span;
    const bool counts = a.tokens != nullptr, biases = a.bias_offsets && a.bias_count;
    const T* x = logits + (int64_t)r * n + i0;
    T* y = out + (int64_t)r * n + i0;
    const uint8_t* mask = a.mask ? reinterpret_cast<const uint8_t*>(a.mask + (int64_t)r * a.mask_stride) + i0 / 8 : nullptr;
    // the logits (and mask) are on their way while the tokens are counted: as whole registers and, where the
    // thread has no 8 of its own, those of another, so that nothing has to wait for them here
    constexpr int NR = (int)sizeof(T) / 2;
    typedef u4 __attribute__((aligned(2))) u4t;
    u4 raw[NR];
    uint32_t bits = 0xFF;
    if (len >= 8) {
        const u4t* from = reinterpret_cast<const u4t*>(x + (tid * 8 + 8 <= len ? tid * 8 : 0));
#pragma unroll
        for (int k = 0; k < NR; k++) raw[k] = from[k];
    }
    if (mask) bits = mask[tid * 8 < len ? tid : 0];
    const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
                pr = a.presence ? a.presence[r] : 0.0f;
    int32_t total = 0, prompt = 0;
    if (counts) {
        total = a.token_counts[r] < (int64_t)a.token_stride ? a.token_counts[r] : (int32_t)a.token_stride;
        prompt = a.prompt_counts ? a.prompt_counts[r] : 0;
    }
    int64_t e0 = 0, e1 = 0;
    if (biases) {
        e0 = a.bias_offsets[r] > 0 ? a.bias_offsets[r] : 0;
        e1 = a.bias_offsets[r + 1] < (int64_t)a.bias_count ? a.bias_offsets[r + 1] : (int64_t)a.bias_count;
    }
    const int32_t* t = a.tokens + (int64_t)r * a.token_stride;
    Some<int32_t, 4> early{{-1, -1, -1, -1}};  // the thread's first tokens, too
    if (tid * 4 + 4 <= total) early = *reinterpret_cast<const Some<int32_t, 4>*>(t + tid * 4);
    if (counts)
        for (int32_t i = tid * 4; i < span; i += 4 * threads) *reinterpret_cast<u4*>(cnt + i) = u4{};
    if (biases)
        for (int32_t i = tid * 4; i < span; i += 4 * threads) *reinterpret_cast<u4*>(entry + i) = ~u4{};
    __syncthreads();
    auto count = [&](int32_t token, int32_t j) {
        const uint32_t i = (uint32_t)token - (uint32_t)i0;
        if (token >= 0 && i < (uint32_t)len) {
            atomicOr(&cnt[i], 0x80000000u);
            if (j >= prompt) atomicAdd(&cnt[i], 1u);
        }
    };
    for (int32_t j = tid * 4; j < total; j += 4 * threads) {
        if (j + 4 <= total) {
            const Some<int32_t, 4> w = j == tid * 4 ? early : *reinterpret_cast<const Some<int32_t, 4>*>(t + j);
#pragma unroll
            for (int k = 0; k < 4; k++) count(w.v[k], j + k);
        } else {
            for (int32_t k = j; k < total; k++) count(t[k], k);
        }
    }
    for (int64_t e = e0 + tid; e < e1; e += threads) {
        const uint32_t i = (uint32_t)a.bias_ids[e] - (uint32_t)i0;
        if (a.bias_ids[e] >= 0 && i < (uint32_t)len) atomicMax(&entry[i], (int32_t)e);
    }
    __syncthreads();
    auto rule = [&](float z, uint32_t c, int32_t e, bool allowed) {
        if (c) {
            z = z > 0.0f ? z / rep : z * rep;
            if (c & 0x7FFFFFFFu) z = z - fr * (float)(c & 0x7FFFFFFFu) - pr;
        }
        if (e >= 0) z += a.bias_values[e];
        return allowed ? z : -INFINITY;
    };
    const bool apart = out != logits;
    const int32_t j = tid * 8;
    if (j + 8 <= len) {
        Some<T, 8> v;
        __builtin_memcpy(&v, raw, sizeof(v));
        uint32_t c[8] = {};
        int32_t e[8] = {-1, -1, -1, -1, -1, -1, -1, -1};
        uint32_t any = 0;
        if (counts) {
#pragma unroll
            for (int k = 0; k < 8; k++) any |= c[k] = cnt[j + k];
        }
        if (biases) {
#pragma unroll
            for (int k = 0; k < 8; k++) any |= ~(uint32_t)(e[k] = entry[j + k]);
        }
        if (any) {
#pragma unroll
            for (int k = 0; k < 8; k++) v.v[k] = (T)rule((float)v.v[k], c[k], e[k], true);
        }
        if (bits != 0xFF) {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (!(bits >> k & 1)) v.v[k] = (T)-INFINITY;
        }
        if (apart || any || bits != 0xFF) *reinterpret_cast<Some<T, 8>*>(y + j) = v;
    } else {
        for (int32_t k = j; k < len; k++) {
            const bool allowed = !mask || mask[k / 8] >> (k % 8) & 1;
            y[k] = (T)rule((float)x[k], counts ? cnt[k] : 0, biases ? entry[k] : -1, allowed);
        }
    }
}

}  // namespace

int launch_logits_rules(void* out, const void* logits, const vvh_logits_spec& r, int64_t rows, int64_t n, int dtype,
                        int64_t cus, void* stream)
{
    // Every block of a row reads the row's whole history and biases: as many threads (and logits) a block as leave
    // two blocks a CU.  A CU holds 2048 threads, whose counters and entries are 128 KB of LDS, in any case.
    int64_t threads = 1024;
    while (threads > 256 && rows * ((n + 8 * threads - 1) / (8 * threads)) < 2 * cus) threads /= 2;
    const int64_t span = 8 * threads;
    const size_t lds = (size_t)span * (r.bias_offsets && r.bias_count ? 8 : r.tokens ? 4 : 0);
    const dim3 grid((unsigned)((n + span - 1) / span), (unsigned)rows);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == VVH_F16)
        hipLaunchKernelGGL(k_logits_rules<f16>, grid, dim3((unsigned)threads), lds, s, (f16*)out, (const f16*)logits, r, (int32_t)n);
    else
        hipLaunchKernelGGL(k_logits_rules<float>, grid, dim3((unsigned)threads), lds, s, (float*)out, (const float*)logits, r, (int32_t)n);
    return (int)hipGetLastError();
}

}  // namespace vvh
