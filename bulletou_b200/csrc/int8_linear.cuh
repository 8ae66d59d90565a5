// Shared by the 8-bit dense layer's kernels (int8_linear.cu, int8_mma.cu).
#pragma once

#include "device_matrix.cuh"

namespace bou {

// out[m][n] = (sum_k q[m][k] w[n][k]) * (scales[m] * w_scales[n]) + bias[n]
struct ProductArgs {
    const int8_t* q;
    const int8_t* w;
    size_t q_stride, w_stride;
    const float* scales;
    const float* w_scales;
    const float* bias;  // null: none
    void* out;
    size_t out_stride;
    int m, n, k;
};

// Every kernel ends in this expression, so a row's results do not depend on
// which of them computed it: one rounding each for the sum's conversion, the
// scales' product and the last operation.
__device__ __forceinline__ float int8_result(int sum, float row_scale, float column_scale, float bias) {
    return __fmaf_rn(static_cast<float>(sum), row_scale * column_scale, bias);
}

// The product on the tensor cores; q and w as a TMA can read them (16-byte
// aligned base and row stride).  `after_quantise`: the launch directly before
// this one on the stream is quantize_kernel, which lets it start early;
// `weights_ready`: that launch does not write the weights.
int launch_int8_mma(BulletOuCudaCppContext* ctx, const ProductArgs& a, int out_type, bool after_quantise, bool weights_ready);

}  // namespace bou
