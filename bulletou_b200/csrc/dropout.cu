// Dropout from a counter-based generator (sm_100a): y = x * [kept] * f (+ r).
//
// The mask is a function of (seed, offset, element index), so the backward
// pass, a second call and any launch shape see the same one and none is kept.
// Generator: Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011).  A block of 128 bits serves
// eight elements with 16 bits each, because the integer work is what could
// bound bf16 rows.  The threshold T = round(p * 2^16) is the probability that
// is used, and f = 2^16 / (2^16 - T), so E[y] = x holds exactly.
//
// Aligned rows are bound by memory: 655360 x 256 bf16 with a residual take 152 to
// 164 us, 6.2 to 6.6 TB/s (a copy: 6.5).  Unaligned ones by instructions: 20011 x 769
// f32 out of rows of 800 take 31 us, 3.9 TB/s, 228 instructions for each piece of up
// to 224 elements.  The generator is the smaller part of them (aligned rows go
// through twice the elements in a time with the same rounds); the rest are
// ballots, selects, and a load and a store for each element of a lane.
#include <algorithm>
#include <cmath>

#include "device_matrix.cuh"
#include "token_launch.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;  // elements of one Philox block
constexpr int kCtas = 4;   // CTAs on an SM: 64 registers for each thread

constexpr int kRounds = 10;

struct Philox {
    uint32_t w[4];
};

struct PhiloxKeys {
    uint2 offset;
    uint2 round[kRounds];  // the key of each round
};

PhiloxKeys philox_keys(uint64_t seed, uint64_t offset) {
    PhiloxKeys k{};
    k.offset = make_uint2(static_cast<uint32_t>(offset), static_cast<uint32_t>(offset >> 32));
    for (uint32_t r = 0; r < kRounds; ++r)
        k.round[r] = make_uint2(static_cast<uint32_t>(seed) + 0x9e3779b9u * r, static_cast<uint32_t>(seed >> 32) + 0xbb67ae85u * r);
    return k;
}

__device__ __forceinline__ Philox philox_block(uint64_t block, const PhiloxKeys& k) {
    uint32_t x0 = static_cast<uint32_t>(block), x1 = static_cast<uint32_t>(block >> 32), x2 = k.offset.x, x3 = k.offset.y;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const uint64_t a = static_cast<uint64_t>(0xd2511f53u) * x0;
        const uint64_t b = static_cast<uint64_t>(0xcd9e8d57u) * x2;
        x0 = static_cast<uint32_t>(b >> 32) ^ x1 ^ k.round[r].x;
        x1 = static_cast<uint32_t>(b);
        x2 = static_cast<uint32_t>(a >> 32) ^ x3 ^ k.round[r].y;
        x3 = static_cast<uint32_t>(a);
    }
    return {{x0, x1, x2, x3}};
}

struct DropoutArgs {
    const void* x;
    const void* residual;
    void* out;
    size_t n;                         // elements
    size_t cols;
    bool flat;                        // no gaps between the rows of any operand
    size_t x_stride, residual_stride, out_stride;
    PhiloxKeys keys;
    uint32_t most_dropped;            // (T << 16) - 1: 16 bits below T, with whatever bits below them
    bool keep_all;                    // T == 0
    float factor;
};

// Lane j (16 bits) is not below T: compared in the upper half of a word, where the
// odd lanes are already and a multiplication brings the even ones.
__device__ __forceinline__ bool kept(const DropoutArgs& a, const Philox& r, int j) {
    return a.keep_all || (j & 1 ? r.w[j >> 1] : r.w[j >> 1] << 16) > a.most_dropped;
}

// Eight neighbouring elements as 16 bytes of bf16 or 32 bytes of f32.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    uint32_t raw[8];
    __device__ __forceinline__ void load(const float* p) {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]),
                       "=r"(raw[7])
                     : "l"(p));
    }
    __device__ __forceinline__ void store(float* p) const {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(raw[0]), "r"(raw[1]),
                     "r"(raw[2]), "r"(raw[3]), "r"(raw[4]), "r"(raw[5]), "r"(raw[6]), "r"(raw[7])
                     : "memory");
    }
    __device__ __forceinline__ float get(int j) const { return __uint_as_float(raw[j]); }
    __device__ __forceinline__ void set(int j, float v) { raw[j] = __float_as_uint(v); }
};
template <>
struct Eight<__nv_bfloat16> {
    __nv_bfloat16 e[8];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        *reinterpret_cast<uint4*>(e) = __ldcs(reinterpret_cast<const uint4*>(p));
    }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const {
        __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(e));
    }
    __device__ __forceinline__ float get(int j) const { return __bfloat162float(e[j]); }
    __device__ __forceinline__ void set(int j, float v) { e[j] = __float2bfloat16_rn(v); }
};

// Rows whose eights are aligned, or (kFlat) one vector: a thread takes the eight
// elements of a block, kBlocks of them with their loads in flight while the
// Philox rounds run.
template <typename T, bool kResidual, bool kFlat>
__global__ void __launch_bounds__(kThreads, kCtas) dropout_vector_kernel(const DropoutArgs a) {
    constexpr int kBlocks = sizeof(T) == 2 ? 2 : 1;
    const size_t blocks = a.n / kLanes, step = static_cast<size_t>(gridDim.x) * kThreads;
    for (size_t b0 = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; b0 < blocks; b0 += step * kBlocks) {
        Eight<T> x[kBlocks], r[kBlocks];
        T* out[kBlocks];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const size_t e = (b0 + i * step) * kLanes;
            const size_t row = kFlat ? 0 : e / a.cols, col = kFlat ? e : e - row * a.cols;
            out[i] = static_cast<T*>(a.out) + row * a.out_stride + col;
            if (b0 + i * step < blocks) {
                x[i].load(static_cast<const T*>(a.x) + row * a.x_stride + col);
                if (kResidual) r[i].load(static_cast<const T*>(a.residual) + row * a.residual_stride + col);
            }
        }
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
            const size_t b = b0 + i * step;
            if (b >= blocks) break;
            const Philox random = philox_block(b, a.keys);
#pragma unroll
            for (int j = 0; j < kLanes; ++j) {
                const float v = kept(a, random, j) ? x[i].get(j) : 0.0f;
                x[i].set(j, kResidual ? __fmaf_rn(v, a.factor, r[i].get(j)) : v * a.factor);
            }
            x[i].store(out[i]);
        }
    }
    // the last elements of a flat vector
    if (kFlat && blockIdx.x == 0 && threadIdx.x < a.n - blocks * kLanes) {
        const size_t e = blocks * kLanes + threadIdx.x;
        const Philox random = philox_block(blocks, a.keys);
        const float v = kept(a, random, threadIdx.x) ? to_f32(static_cast<const T*>(a.x)[e]) : 0.0f;
        static_cast<T*>(a.out)[e] = from_f32<T>(kResidual ? __fmaf_rn(v, a.factor, to_f32(static_cast<const T*>(a.residual)[e]))
                                                          : v * a.factor);
    }
}

// Rows of any stride and alignment, wide ones: a warp takes pieces of 7 x 32
// elements of a row, whose blocks its 32 lanes can compute wherever the piece
// begins inside a block.  The lanes' decisions on each block's k-th element make
// one word; a lane's elements are all the k-th of their blocks, 4 blocks apart,
// so it picks its word once and tests a bit for each element.  The elements are
// read and written 32 neighbours at a time.
constexpr int kTurns = 7;
constexpr int kPiece = kTurns * 32;
constexpr int kWideRow = 64;  // columns from which a piece fills most of a warp's turns
template <bool kResidual>
constexpr int kRowCtas = kResidual ? 4 : 6;

template <bool kFull, typename T, bool kResidual>
__device__ __forceinline__ void dropout_piece(const DropoutArgs& a, size_t row, size_t col, int count) {
    const int lane = threadIdx.x & 31;
    const T* const x_at = static_cast<const T*>(a.x) + row * a.x_stride + col + lane;
    const T* const r_at = kResidual ? static_cast<const T*>(a.residual) + row * a.residual_stride + col + lane : nullptr;
    T* const out = static_cast<T*>(a.out) + row * a.out_stride + col + lane;
    const int left = count - lane;
    T x[kTurns], r[kTurns];
#pragma unroll
    for (int j = 0; j < kTurns; ++j)
        if (kFull || j * 32 < left) {
            x[j] = x_at[j * 32];
            if (kResidual) r[j] = r_at[j * 32];
        }
    const size_t element = row * a.cols + col;
    const Philox random = philox_block(element / kLanes + lane, a.keys);
    const int place = static_cast<int>(element % kLanes) + lane;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < kLanes; ++k) {
        const uint32_t decisions = __ballot_sync(0xffffffffu, kept(a, random, k));
        if ((place & (kLanes - 1)) == k) word = decisions;
    }
    word >>= place / kLanes;
#pragma unroll
    for (int j = 0; j < kTurns; ++j)
        if (kFull || j * 32 < left) {
            const float v = word & (1u << (4 * j)) ? to_f32(x[j]) : 0.0f;
            out[j * 32] = from_f32<T>(kResidual ? __fmaf_rn(v, a.factor, to_f32(r[j])) : v * a.factor);
        }
}

template <typename T, bool kResidual>
__global__ void __launch_bounds__(kThreads, kRowCtas<kResidual>) dropout_row_kernel(const DropoutArgs a, int pieces) {
    const size_t rows = a.n / a.cols, step = static_cast<size_t>(gridDim.x) * (kThreads / 32);
    for (size_t row = static_cast<size_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); row < rows; row += step)
        for (int s = blockIdx.y; s < pieces; s += gridDim.y) {
            const size_t col = static_cast<size_t>(s) * kPiece;
            if (a.cols - col >= kPiece) dropout_piece<true, T, kResidual>(a, row, col, kPiece);
            else dropout_piece<false, T, kResidual>(a, row, col, static_cast<int>(a.cols - col));
        }
}

// Narrow rows of any stride and alignment: a warp takes 32 blocks, that is 256
// elements in row-major order over as many rows as they are.
template <typename T, bool kResidual>
__global__ void __launch_bounds__(kThreads, kCtas) dropout_kernel(const DropoutArgs a) {
    const int lane = threadIdx.x & 31;
    const size_t blocks = (a.n + kLanes - 1) / kLanes;
    // 32 elements further on: so many rows and columns, and what a full row's end adds
    const uint32_t cols = static_cast<uint32_t>(a.cols), rows32 = 32 / cols, cols32 = 32 % cols;
    const size_t x_step = rows32 * a.x_stride + cols32, x_wrap = a.x_stride - cols;
    const size_t r_step = rows32 * a.residual_stride + cols32, r_wrap = a.residual_stride - cols;
    const size_t out_step = rows32 * a.out_stride + cols32, out_wrap = a.out_stride - cols;
    for (size_t b0 = static_cast<size_t>(blockIdx.x) * kThreads + (threadIdx.x & ~31); b0 < blocks;
         b0 += static_cast<size_t>(gridDim.x) * kThreads) {
        const size_t e = b0 * kLanes + lane, row = e / cols;
        uint32_t col = static_cast<uint32_t>(e - row * cols);
        const int left = static_cast<int>(a.n - b0 * kLanes < 256 ? a.n - b0 * kLanes : 256);
        const T* x_at = static_cast<const T*>(a.x) + row * a.x_stride + col;
        const T* r_at = kResidual ? static_cast<const T*>(a.residual) + row * a.residual_stride + col : nullptr;
        float x[kLanes], r[kLanes];
        uint32_t wraps = 0;  // bit j: element j is followed by a row's end
#pragma unroll
        for (int j = 0; j < kLanes; ++j) {
            const bool in = j * 32 + lane < left;
            x[j] = in ? to_f32(*x_at) : 0.0f;
            if (kResidual) r[j] = in ? to_f32(*r_at) : 0.0f;
            col += cols32;
            const bool wrap = col >= cols;
            if (wrap) col -= cols;
            wraps |= wrap ? 1u << j : 0u;
            x_at += x_step + (wrap ? x_wrap : 0);
            if (kResidual) r_at += r_step + (wrap ? r_wrap : 0);
        }
        const Philox random = philox_block(b0 + lane, a.keys);
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < kLanes; ++j) mask |= kept(a, random, j) ? 1u << j : 0u;
        T* out = static_cast<T*>(a.out) + row * a.out_stride + (e - row * cols);
#pragma unroll
        for (int j = 0; j < kLanes; ++j) {
            const uint32_t theirs = __shfl_sync(0xffffffffu, mask, j * 4 + (lane >> 3));
            const float v = (theirs >> (lane & 7)) & 1u ? x[j] : 0.0f;
            if (j * 32 + lane < left) *out = from_f32<T>(kResidual ? __fmaf_rn(v, a.factor, r[j]) : v * a.factor);
            out += out_step + ((wraps >> j) & 1u ? out_wrap : 0);
        }
    }
}

template <typename T, bool kResidual>
int launch_dropout(BulletOuCudaCppContext* ctx, const DropoutArgs& a, bool vector) {
    const int64_t per_cta = static_cast<int64_t>(kThreads) * kLanes;
    const int64_t ctas = (static_cast<int64_t>(a.n) + per_cta - 1) / per_cta;
    const LaunchShape shape{dim3(static_cast<unsigned>(std::min<int64_t>(ctas, ctx->sm_count * kCtas))), kThreads};
    if (!vector && a.cols >= kWideRow) {
        const int64_t rows = static_cast<int64_t>(a.n / a.cols), row_ctas = (rows + kThreads / 32 - 1) / (kThreads / 32);
        const int pieces = static_cast<int>((a.cols + kPiece - 1) / kPiece);
        const int64_t resident = static_cast<int64_t>(ctx->sm_count) * kRowCtas<kResidual>;
        const unsigned x = static_cast<unsigned>(std::min(row_ctas, resident));
        const unsigned y = static_cast<unsigned>(std::min<int64_t>(pieces, std::max<int64_t>(1, resident / x)));
        return launch_kernel(ctx, "dropout launch", dropout_row_kernel<T, kResidual>, LaunchShape{dim3(x, y), kThreads}, a, pieces);
    }
    if (!vector) return launch_kernel(ctx, "dropout launch", dropout_kernel<T, kResidual>, shape, a);
    if (a.flat) return launch_kernel(ctx, "dropout launch", dropout_vector_kernel<T, kResidual, true>, shape, a);
    return launch_kernel(ctx, "dropout launch", dropout_vector_kernel<T, kResidual, false>, shape, a);
}

template <typename T>
int launch_dropout(BulletOuCudaCppContext* ctx, const DropoutArgs& a, bool vector) {
    return a.residual != nullptr ? launch_dropout<T, true>(ctx, a, vector) : launch_dropout<T, false>(ctx, a, vector);
}

}  // namespace
}  // namespace bou

using namespace bou;

extern "C" {

int bulletou_b200_dropout_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* x,
                                 const BulletOuB200Matrix* residual, double probability, unsigned long long seed,
                                 unsigned long long offset, const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(x, kTypeFloat, "dropout x") != 0) return -1;
    const unsigned type = 1u << x->type;
    if (validate_matrix(out, type, x->rows, x->cols, "dropout out") != 0 ||
        (residual != nullptr && validate_matrix(residual, type, x->rows, x->cols, "dropout residual") != 0) ||
        validate_disjoint(out, "dropout out", x, "x", true) != 0 ||
        validate_disjoint(out, "dropout out", residual, "residual", true) != 0)
        return -1;
    if (!(probability >= 0.0 && probability <= 1.0))
        return fail_messagef("dropout probability must be in [0, 1], got %g", probability);
    DropoutArgs a{};
    a.n = x->rows * x->cols;
    if (a.n == 0) return ok();
    a.x = x->data;
    a.residual = residual != nullptr ? residual->data : nullptr;
    a.out = out->data;
    a.cols = x->cols;
    a.x_stride = x->row_stride;
    a.residual_stride = residual != nullptr ? residual->row_stride : 0;
    a.out_stride = out->row_stride;
    a.keys = philox_keys(seed, offset);
    const uint32_t threshold = static_cast<uint32_t>(std::floor(probability * 65536.0 + 0.5));
    a.keep_all = threshold == 0;
    a.most_dropped = static_cast<uint32_t>((static_cast<uint64_t>(threshold) << 16) - 1);  // 65536: every word
    a.factor = threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - threshold)) : 0.0f;
    // a vector where every eight is aligned: rows of whole eights, or no gaps between rows at all
    a.flat = is_flat(*x) && is_flat(*out) && (residual == nullptr || is_flat(*residual));
    const size_t unit = kLanes * type_bytes(x->type);
    auto aligned = [&](const BulletOuB200Matrix& m) {
        return a.flat ? reinterpret_cast<uintptr_t>(m.data) % unit == 0 : rows_aligned(m, unit);
    };
    const bool vector = (a.flat || x->cols % kLanes == 0) && aligned(*x) && aligned(*out) && (residual == nullptr || aligned(*residual));
    const int rc = x->type == BULLETOU_B200_TYPE_F32 ? launch_dropout<float>(ctx, a, vector)
                                                     : launch_dropout<__nv_bfloat16>(ctx, a, vector);
    return rc != 0 ? rc : ok();
}

}  // extern "C"
