// q4.hip — products of rows with weights in 4 bits.
#include <hip/hip_runtime.h>

#include "device.hpp"
#include "drafts.hpp"

namespace m1moe {

namespace {

// y[t][n] = sum_k x[t][k] (q[n][k] s[n][k / G] + b[n][k / G]) (+ r[t][n]): a wave per (n, t).
template <bool XB>
__global__ __launch_bounds__(256) void q4_simple_kernel(Q4Args a) {
    const int lane = threadIdx.x & 63, t = (int)blockIdx.y;
    const int n = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= a.rows) return;
    const int words = a.cols / 8, groups = a.cols / a.group;
    float sum = 0.f;
    for (int w = lane; w < words; w += 64) {
        const uint32_t q = a.w[(int64_t)n * words + w];
        const int64_t g = (int64_t)n * groups + 8 * w / a.group;
        const float s = bf16_to_f32(a.scales[g]), b = bf16_to_f32(a.biases[g]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t at = (int64_t)t * a.x_stride + 8 * w + j;
            const float x = XB ? bf16_to_f32(static_cast<const uint16_t*>(a.x)[at]) : static_cast<const float*>(a.x)[at];
            sum = fmaf(x, fmaf((float)(q >> 4 * j & 15), s, b), sum);
        }
    }
    sum = wave_sum(sum);
    if (lane) return;
    const int64_t at = (int64_t)t * a.y_stride + n;
    if (a.y_bf16) {
        if (a.residual) sum += bf16_to_f32(static_cast<const uint16_t*>(a.residual)[at]);
        static_cast<__bf16*>(a.y)[at] = (__bf16)sum;
    } else {
        if (a.residual) sum += static_cast<const float*>(a.residual)[at];
        static_cast<float*>(a.y)[at] = sum;
    }
}

}  // namespace

int launch_matmul_q4(const Q4Args& a, int, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)((a.rows + 3) / 4), (unsigned)a.tokens);
    if (a.x_bf16)
        hipLaunchKernelGGL(q4_simple_kernel<true>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(q4_simple_kernel<false>, grid, dim3(256), 0, st, a);
    return (int)hipGetLastError();
}

}  // namespace m1moe
