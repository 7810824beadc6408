// Linears of 4-bit weights with group scales:
//   out[m][n] = sum_g s[n][g] sum_{k in g} (c[n][k] - z[n][g]) x[m][k] + bias[n] + res[m][n]
// with the codes c two to a byte, scales s in fp16 and zero points z bytes (8
// where there are none).
#include <hip/hip_runtime.h>

#include "common.h"
#include "device.h"

namespace vvh {

namespace {

// One wave per output channel: lane l takes the 8 codes of dword l, l + 64, ... of
// the weight row (one group: groups are whole dwords) for up to 8 rows of x.
template <typename T, typename OT>
__global__ __launch_bounds__(256) void k_linear_q4(Q4Args a)
{
    const int lane = threadIdx.x & 63;
    const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= a.N) return;
    const int64_t groups = a.K / a.group;
    for (int64_t m0 = 0; m0 < a.M; m0 += 8) {
        float acc[8] = {};
        for (int64_t k = lane * 8; k < a.K; k += 512) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(a.w + (n * a.K + k) / 2);
            const int64_t g = n * groups + k / a.group;
            const float s = (float)reinterpret_cast<const f16*>(a.scales)[g], z = a.zeros ? (float)a.zeros[g] : 8.0f;
#pragma unroll
            for (int m = 0; m < 8; m++) {
                if (m0 + m >= a.M) break;
                const T* x = (const T*)a.inp + (m0 + m) * a.K + k;
                float d = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) d = __builtin_fmaf((float)((w >> (4 * j)) & 15) - z, (float)x[j], d);
                acc[m] = __builtin_fmaf(s, d, acc[m]);
            }
        }
#pragma unroll
        for (int m = 0; m < 8; m++) {
            const float y = wave_sum_xor(acc[m]);
            if (lane == 0 && m0 + m < a.M) {
                const int64_t o = (m0 + m) * a.N + n;
                ((OT*)a.out)[o] = (OT)(y + (a.bias ? a.bias[n] : 0.0f) + (a.res ? (float)((const OT*)a.res)[o] : 0.0f));
            }
        }
    }
}

}  // namespace

int launch_linear_q4(const Q4Args& a, int act, int out, void* stream)
{
    const dim3 grid((unsigned)((a.N + 3) / 4));
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a); };
    if (act == VVH_F16) out == VVH_F16 ? go(k_linear_q4<f16, f16>) : go(k_linear_q4<f16, float>);
    else out == VVH_F16 ? go(k_linear_q4<float, f16>) : go(k_linear_q4<float, float>);
    return (int)hipGetLastError();
}

}  // namespace vvh
