// Dropout from a counter-based generator (sm_100a): y = x * [kept] * f (+ r).
//
// The mask is a function of (seed, offset, element index), so the backward
// pass, a second call and any launch shape see the same one and none is kept.
// Generator: Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  A block of 128 bits serves
// eight elements with 16 bits each, because the integer work is what could
// bound bf16 rows.  The threshold T = round(p * 2^16) is the probability that
// is used, and f = 2^16 / (2^16 - T), so E[y] = x holds exactly.
#include <algorithm>
#include <cmath>

#include "device_matrix.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;  // elements of one Philox block

struct Philox {
    uint32_t w[4];
};

__device__ __forceinline__ Philox philox_block(uint64_t block, uint2 offset, uint2 key) {
    uint32_t x0 = static_cast<uint32_t>(block), x1 = static_cast<uint32_t>(block >> 32), x2 = offset.x, x3 = offset.y;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = static_cast<uint64_t>(0xd2511f53u) * x0;
        const uint64_t b = static_cast<uint64_t>(0xcd9e8d57u) * x2;
        const uint32_t k0 = key.x + 0x9e3779b9u * r, k1 = key.y + 0xbb67ae85u * r;
        x0 = static_cast<uint32_t>(b >> 32) ^ x1 ^ k0;
        x1 = static_cast<uint32_t>(b);
        x2 = static_cast<uint32_t>(a >> 32) ^ x3 ^ k1;
        x3 = static_cast<uint32_t>(a);
    }
    return {{x0, x1, x2, x3}};
}

struct DropoutArgs {
    const void* x;
    const void* residual;
    void* out;
    size_t n;                         // elements
    uint32_t cols;
    size_t x_stride, residual_stride, out_stride;
    uint2 key, offset;
    uint32_t threshold;               // dropped below; 65536: everything
    float factor;
};

// A thread takes the eight elements of one block.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const DropoutArgs a) {
    const size_t blocks = (a.n + kLanes - 1) / kLanes;
    for (size_t b = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; b < blocks;
         b += static_cast<size_t>(gridDim.x) * kThreads) {
        const Philox r = philox_block(b, a.offset, a.key);
        size_t row = b * kLanes / a.cols;
        uint32_t col = static_cast<uint32_t>(b * kLanes - row * a.cols);
#pragma unroll
        for (int j = 0; j < kLanes; ++j) {
            if (b * kLanes + j >= a.n) break;
            const uint32_t u = (r.w[j >> 1] >> (16 * (j & 1))) & 0xffffu;
            const bool kept = u >= a.threshold;
            float y = kept ? to_f32(static_cast<const T*>(a.x)[row * a.x_stride + col]) * a.factor : 0.0f;
            if (a.residual != nullptr) y += to_f32(static_cast<const T*>(a.residual)[row * a.residual_stride + col]);
            static_cast<T*>(a.out)[row * a.out_stride + col] = from_f32<T>(y);
            if (++col == a.cols) {
                col = 0;
                ++row;
            }
        }
    }
}

}  // namespace
}  // namespace bou

using namespace bou;

extern "C" {

int bulletou_b200_dropout_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* x,
                                 const BulletOuB200Matrix* residual, float probability, unsigned long long seed,
                                 unsigned long long offset, const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(x, kTypeFloat, "dropout x") != 0) return -1;
    const unsigned type = 1u << x->type;
    if (validate_matrix(out, type, x->rows, x->cols, "dropout out") != 0 ||
        (residual != nullptr && validate_matrix(residual, type, x->rows, x->cols, "dropout residual") != 0) ||
        validate_disjoint(out, "dropout out", x, "x", true) != 0 ||
        validate_disjoint(out, "dropout out", residual, "residual", true) != 0)
        return -1;
    if (!(probability >= 0.0f && probability <= 1.0f))
        return fail_messagef("dropout probability must be in [0, 1], got %g", static_cast<double>(probability));
    DropoutArgs a{};
    a.n = x->rows * x->cols;
    if (a.n == 0) return ok();
    a.x = x->data;
    a.residual = residual != nullptr ? residual->data : nullptr;
    a.out = out->data;
    a.cols = static_cast<uint32_t>(x->cols);
    a.x_stride = x->row_stride;
    a.residual_stride = residual != nullptr ? residual->row_stride : 0;
    a.out_stride = out->row_stride;
    a.key = make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
    a.offset = make_uint2(static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32));
    a.threshold = static_cast<uint32_t>(std::floor(static_cast<double>(probability) * 65536.0 + 0.5));
    a.factor = a.threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - a.threshold)) : 0.0f;
    const size_t blocks = (a.n + kLanes * kThreads - 1) / (kLanes * kThreads);
    const int grid = static_cast<int>(std::min<size_t>(blocks, static_cast<size_t>(ctx->sm_count) * 8));
    if (x->type == BULLETOU_B200_TYPE_F32)
        dropout_kernel<float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else
        dropout_kernel<__nv_bfloat16><<<grid, kThreads, 0, ctx->stream>>>(a);
    return check_launch("dropout launch") != 0 ? -1 : ok();
}

}  // extern "C"
