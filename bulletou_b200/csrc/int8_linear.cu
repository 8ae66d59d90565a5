// Dense layer in 8-bit integers with a scale for each token (row) and each
// output channel (sm_100a).
//
//   s_m = max_k |x_mk| * (1/127),   q_mk = rint(x_mk * (127 * (1 / max_k |x_mk|)))
//   y_mn = (sum_k q_mk w_nk) * (s_m * w_scale_n) + bias_n
// The sum is exact in 32-bit integers for K <= 131072 (127^2 K < 2^31), so it
// may be cut and joined in any order.
#include <algorithm>
#include <cmath>

#include "device_matrix.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ quantisation
struct QuantizeArgs {
    const void* x;
    size_t x_stride;
    int8_t* q;
    size_t q_stride;
    float* scales;
    int cols, padded_cols;  // columns [cols, padded_cols) of q are zeroed
};

// CTA per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeArgs a) {
    __shared__ float warp_top[kThreads / 32];
    const T* x = static_cast<const T*>(a.x) + blockIdx.x * a.x_stride;
    int8_t* q = a.q + blockIdx.x * a.q_stride;
    float top = 0.0f;
    bool bad = false;
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
        const float v = fabsf(to_f32(x[c]));
        bad |= !(v < INFINITY);
        top = fmaxf(top, v);
    }
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, warp_top[w]);
    const bool some = !bad && top >= 0x1p-100f;
    const float inverse = some ? 127.0f * __frcp_rn(top) : 0.0f;
    for (int c = threadIdx.x; c < a.padded_cols; c += kThreads)
        q[c] = c < a.cols && some ? static_cast<int8_t>(__float2int_rn(to_f32(x[c]) * inverse)) : 0;
    if (threadIdx.x == 0) a.scales[blockIdx.x] = bad ? NAN : some ? top * (1.0f / 127.0f) : 0.0f;
}

// ------------------------------------------------------------------ product
struct ProductArgs {
    const int8_t* q;
    const int8_t* w;
    size_t q_stride, w_stride;
    const float* scales;
    const float* w_scales;
    const float* bias;
    void* out;
    size_t out_stride;
    int m, n, k;
};

constexpr int kTileM = 64, kTileN = 64, kTileK = 64;

// A 64 x 64 tile of the output, 4 x 4 results for each thread.
template <typename Out>
__global__ void __launch_bounds__(kThreads) product_kernel(const ProductArgs a) {
    __shared__ int sq[kTileK / 4][kTileM + 1], sw[kTileK / 4][kTileN + 1];
    const int m0 = blockIdx.y * kTileM, n0 = blockIdx.x * kTileN;
    const int tm = (threadIdx.x >> 4) * 4, tn = (threadIdx.x & 15) * 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += kTileK) {
        for (int i = threadIdx.x; i < kTileM * kTileK; i += kThreads) {
            const int r = i / kTileK, c = i % kTileK;
            const bool k_in = k0 + c < a.k;
            reinterpret_cast<int8_t*>(&sq[c / 4][r])[c % 4] =
                k_in && m0 + r < a.m ? a.q[static_cast<size_t>(m0 + r) * a.q_stride + k0 + c] : 0;
            reinterpret_cast<int8_t*>(&sw[c / 4][r])[c % 4] =
                k_in && n0 + r < a.n ? a.w[static_cast<size_t>(n0 + r) * a.w_stride + k0 + c] : 0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kTileK / 4; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sq[c][tm + i], sw[c][tn + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + tm + i, n = n0 + tn + j;
            if (m >= a.m || n >= a.n) continue;
            float y = static_cast<float>(acc[i][j]) * (a.scales[m] * a.w_scales[n]);
            if (a.bias != nullptr) y += a.bias[n];
            static_cast<Out*>(a.out)[static_cast<size_t>(m) * a.out_stride + n] = from_f32<Out>(y);
        }
}

int quantize(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix& x, int8_t* q, size_t q_stride, int padded_cols,
             float* scales) {
    QuantizeArgs a{};
    a.x = x.data;
    a.x_stride = x.row_stride;
    a.q = q;
    a.q_stride = q_stride;
    a.scales = scales;
    a.cols = static_cast<int>(x.cols);
    a.padded_cols = padded_cols;
    const int grid = static_cast<int>(x.rows);
    if (x.type == BULLETOU_B200_TYPE_F32)
        quantize_kernel<float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else
        quantize_kernel<__nv_bfloat16><<<grid, kThreads, 0, ctx->stream>>>(a);
    return check_launch("int8 quantise launch");
}

int product(BulletOuCudaCppContext* ctx, const ProductArgs& a, int out_type) {
    const unsigned gm = (a.m + kTileM - 1) / kTileM;
    if (gm > 65535u) return fail_messagef("int8 product: %d rows are not supported", a.m);
    const dim3 grid((a.n + kTileN - 1) / kTileN, gm);
    if (out_type == BULLETOU_B200_TYPE_F32)
        product_kernel<float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else
        product_kernel<__nv_bfloat16><<<grid, kThreads, 0, ctx->stream>>>(a);
    return check_launch("int8 product launch");
}

// The weight side's checks, shared by the two products.
int validate_weights(const BulletOuB200Matrix* in, const char* in_name, const BulletOuB200Matrix* weights,
                     const BulletOuB200Matrix* weight_scales, const BulletOuB200Matrix* bias,
                     const BulletOuB200Matrix* out) {
    if (validate_matrix(weights, kTypeI8, "int8 weights") != 0) return -1;
    if (in->cols > BULLETOU_B200_INT8_MAX_INNER)
        return fail_messagef("int8: %zu inner columns, at most %d are exact", in->cols, BULLETOU_B200_INT8_MAX_INNER);
    if (validate_matrix(weights, kTypeI8, weights->rows, in->cols, "int8 weights") != 0 ||
        validate_matrix(weight_scales, kTypeF32, 1, weights->rows, "int8 weight scales") != 0 ||
        (bias != nullptr && validate_matrix(bias, kTypeF32, 1, weights->rows, "int8 bias") != 0) ||
        validate_matrix(out, kTypeFloat, in->rows, weights->rows, "int8 out") != 0 ||
        validate_disjoint(out, "int8 out", in, in_name) != 0 ||
        validate_disjoint(out, "int8 out", weights, "the weights") != 0 ||
        validate_disjoint(out, "int8 out", weight_scales, "the weight scales") != 0 ||
        validate_disjoint(out, "int8 out", bias, "the bias") != 0)
        return -1;
    return 0;
}

ProductArgs product_args(const BulletOuB200Matrix& weights, const BulletOuB200Matrix& weight_scales,
                         const BulletOuB200Matrix* bias, const BulletOuB200Matrix& out) {
    ProductArgs a{};
    a.w = static_cast<const int8_t*>(weights.data);
    a.w_stride = weights.row_stride;
    a.w_scales = static_cast<const float*>(weight_scales.data);
    a.bias = bias != nullptr ? static_cast<const float*>(bias->data) : nullptr;
    a.out = out.data;
    a.out_stride = out.row_stride;
    a.m = static_cast<int>(out.rows);
    a.n = static_cast<int>(out.cols);
    a.k = static_cast<int>(weights.cols);
    return a;
}

}  // namespace
}  // namespace bou

using namespace bou;

extern "C" {

int bulletou_b200_int8_quantize_rows_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* x,
                                            const BulletOuB200Matrix* q, const BulletOuB200Matrix* scales) {
    if (set_device(ctx) != 0 || validate_matrix(x, kTypeFloat, "int8 x") != 0 ||
        validate_matrix(q, kTypeI8, x->rows, x->cols, "int8 q") != 0 ||
        validate_matrix(scales, kTypeF32, 1, x->rows, "int8 scales") != 0 ||
        validate_disjoint(q, "int8 q", x, "x") != 0 || validate_disjoint(scales, "int8 scales", x, "x") != 0 ||
        validate_disjoint(scales, "int8 scales", q, "q") != 0)
        return -1;
    if (x->rows == 0) return ok();
    return quantize(ctx, *x, static_cast<int8_t*>(q->data), q->row_stride, static_cast<int>(x->cols),
                    static_cast<float*>(scales->data)) != 0
               ? -1
               : ok();
}

int bulletou_b200_int8_matmul_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* q,
                                     const BulletOuB200Matrix* scales, const BulletOuB200Matrix* weights,
                                     const BulletOuB200Matrix* weight_scales, const BulletOuB200Matrix* bias,
                                     const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(q, kTypeI8, "int8 q") != 0 ||
        validate_matrix(scales, kTypeF32, 1, q->rows, "int8 scales") != 0 ||
        validate_weights(q, "q", weights, weight_scales, bias, out) != 0 ||
        validate_disjoint(out, "int8 out", scales, "the scales") != 0)
        return -1;
    ProductArgs a = product_args(*weights, *weight_scales, bias, *out);
    if (a.m == 0 || a.n == 0) return ok();
    a.q = static_cast<const int8_t*>(q->data);
    a.q_stride = q->row_stride;
    a.scales = static_cast<const float*>(scales->data);
    return product(ctx, a, out->type) != 0 ? -1 : ok();
}

int bulletou_b200_int8_linear_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* x,
                                     const BulletOuB200Matrix* weights, const BulletOuB200Matrix* weight_scales,
                                     const BulletOuB200Matrix* bias, const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(x, kTypeFloat, "int8 x") != 0 ||
        validate_weights(x, "x", weights, weight_scales, bias, out) != 0)
        return -1;
    ProductArgs a = product_args(*weights, *weight_scales, bias, *out);
    if (a.m == 0 || a.n == 0) return ok();
    a.q_stride = (static_cast<size_t>(a.k) + 15) / 16 * 16;
    const size_t scale_bytes = (static_cast<size_t>(a.m) * sizeof(float) + 255) / 256 * 256;
    void* p = nullptr;
    if (scratch_slot(ctx, kScratchInt8, scale_bytes + a.m * a.q_stride, &p, "cudaMalloc int8 rows") != 0) return -1;
    float* const scales = static_cast<float*>(p);
    int8_t* const q = static_cast<int8_t*>(p) + scale_bytes;
    a.scales = scales;
    a.q = q;
    if (quantize(ctx, *x, q, a.q_stride, static_cast<int>(a.q_stride), scales) != 0) return -1;
    return product(ctx, a, out->type) != 0 ? -1 : ok();
}

}  // extern "C"
