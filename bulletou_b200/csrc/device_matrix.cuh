// Matrices in device memory as the token-layer entries take them
// (BulletOuB200Matrix): their checks, and element loads and stores that hold
// every value in f32.
#pragma once

#include <cuda_bf16.h>

#include <cstdint>

#include "common.cuh"

namespace bou {

constexpr unsigned kTypeF32 = 1u << BULLETOU_B200_TYPE_F32;
constexpr unsigned kTypeBf16 = 1u << BULLETOU_B200_TYPE_BF16;
constexpr unsigned kTypeI8 = 1u << BULLETOU_B200_TYPE_I8;
constexpr unsigned kTypeI32 = 1u << BULLETOU_B200_TYPE_I32;
constexpr unsigned kTypeFloat = kTypeF32 | kTypeBf16;

inline size_t type_bytes(int type) {
    return type == BULLETOU_B200_TYPE_I8 ? 1 : type == BULLETOU_B200_TYPE_BF16 ? 2 : 4;
}

// 0 if `m` is a rows x cols matrix of one of `types` (a mask of kType*) that
// can be addressed; the message names it otherwise.
int validate_matrix(const BulletOuB200Matrix* m, unsigned types, size_t rows, size_t cols, const char* name);
// The same without a demand on its extents.
int validate_matrix(const BulletOuB200Matrix* m, unsigned types, const char* name);
// 0 if writing `out` leaves `in` as it was.  `same_ok`: the two may be the very
// same elements (an element-wise operator in place).
int validate_disjoint(const BulletOuB200Matrix* out, const char* out_name, const BulletOuB200Matrix* in,
                      const char* in_name, bool same_ok = false);

// Rows follow one another without a gap, so the matrix is one vector.
inline bool is_flat(const BulletOuB200Matrix& m) { return m.rows <= 1 || m.row_stride == m.cols; }

// Every row starts on a multiple of `bytes`.
inline bool rows_aligned(const BulletOuB200Matrix& m, size_t bytes) {
    return reinterpret_cast<uintptr_t>(m.data) % bytes == 0 &&
           (m.rows <= 1 || m.row_stride * type_bytes(m.type) % bytes == 0);
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace bou
