// The rules between a row of logits and its sampler: penalties of tokens that were
// there before, biases, and a mask of allowed tokens.
#include <hip/hip_runtime.h>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// Logits of a block, and its threads.  Their counters and bias entries are LDS words.
constexpr int kRulesSpan = 2048;

// Block (x, r): logits [x * kRulesSpan, ...) of row r.  It counts the row's
// tokens that fall into its span (bit 31: seen at all; below it the times among
// those after the prompt; sums of integers, so in any order) and finds each
// biased token's last entry, then takes its logits through the rules.
template <typename T>
__global__ __launch_bounds__(256) void k_logits_rules(T* out, const T* logits, vvh_logits_spec a, int32_t n)
{
    __shared__ uint32_t cnt[kRulesSpan];
    __shared__ int32_t entry[kRulesSpan];
    const int32_t r = blockIdx.y, i0 = blockIdx.x * kRulesSpan, tid = threadIdx.x;
    const int32_t span = n - i0 < kRulesSpan ? n - i0 : kRulesSpan;
    for (int32_t i = tid; i < kRulesSpan; i += 256) {
        cnt[i] = 0;
        entry[i] = -1;
    }
    __syncthreads();
    if (a.tokens) {
        const int32_t total = a.token_counts[r] < (int64_t)a.token_stride ? a.token_counts[r] : (int32_t)a.token_stride;
        const int32_t prompt = a.prompt_counts ? a.prompt_counts[r] : 0;
        const int32_t* t = a.tokens + (int64_t)r * a.token_stride;
        for (int32_t j = tid; j < total; j += 256) {
            const uint32_t i = (uint32_t)t[j] - (uint32_t)i0;
            if (t[j] >= 0 && i < (uint32_t)span) {
                atomicOr(&cnt[i], 0x80000000u);
                if (j >= prompt) atomicAdd(&cnt[i], 1u);
            }
        }
    }
    if (a.bias_offsets && a.bias_count) {
        const int64_t e0 = a.bias_offsets[r] > 0 ? a.bias_offsets[r] : 0;
        const int64_t e1 = a.bias_offsets[r + 1] < (int64_t)a.bias_count ? a.bias_offsets[r + 1] : (int64_t)a.bias_count;
        for (int64_t e = e0 + tid; e < e1; e += 256) {
            const uint32_t i = (uint32_t)a.bias_ids[e] - (uint32_t)i0;
            if (a.bias_ids[e] >= 0 && i < (uint32_t)span) atomicMax(&entry[i], (int32_t)e);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[r] : 1.0f, fr = a.frequency ? a.frequency[r] : 0.0f,
                pr = a.presence ? a.presence[r] : 0.0f;
    const uint32_t* mask = a.mask ? a.mask + (int64_t)r * a.mask_stride : nullptr;
    for (int32_t j = tid; j < span; j += 256) {
        const int32_t i = i0 + j;
        const int64_t at = (int64_t)r * n + i;
        float x = (float)logits[at];
        const uint32_t c = cnt[j];
        if (c) {
            x = x > 0.0f ? x / rep : x * rep;
            if (c & 0x7FFFFFFFu) x = x - fr * (float)(c & 0x7FFFFFFFu) - pr;
        }
        if (entry[j] >= 0) x += a.bias_values[entry[j]];
        if (mask && !(mask[i >> 5] >> (i & 31) & 1)) x = -INFINITY;
        out[at] = (T)x;
    }
}

}  // namespace

int launch_logits_rules(void* out, const void* logits, const vvh_logits_spec& r, int64_t rows, int64_t n, int dtype,
                        void* stream)
{
    const dim3 grid((unsigned)((n + kRulesSpan - 1) / kRulesSpan), (unsigned)rows);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == VVH_F16)
        hipLaunchKernelGGL(k_logits_rules<f16>, grid, dim3(256), 0, s, (f16*)out, (const f16*)logits, r, (int32_t)n);
    else
        hipLaunchKernelGGL(k_logits_rules<float>, grid, dim3(256), 0, s, (float*)out, (const float*)logits, r, (int32_t)n);
    return (int)hipGetLastError();
}

}  // namespace vvh
