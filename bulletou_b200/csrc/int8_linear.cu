// Dense layer in 8-bit integers with a scale for each token (row) and each
// output channel (sm_100a).
//
//   s_m = max_k |x_mk| * (1/127),   q_mk = rint(x_mk * (127 * (1 / max_k |x_mk|)))
//   y_mn = (sum_k q_mk w_nk) * (s_m * w_scale_n) + bias_n
// The sum is exact in 32-bit integers for K <= 131071 (128^2 K < 2^31), so it
// may be cut and joined in any order.
#include <algorithm>
#include <cmath>

#include "int8_linear.cuh"
#include "token_launch.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kSmallest = 0x1p-100f;  // rows below it are zeros: 1 / m and 127 / m stay finite

__device__ __forceinline__ float row_factor(float top) { return 127.0f * __frcp_rn(top); }
__device__ __forceinline__ float row_scale(float top) { return top * (1.0f / 127.0f); }
__device__ __forceinline__ int quantised(float x, float factor) { return __float2int_rn(x * factor); }

// ------------------------------------------------------------------ bytes
// A matrix of bytes with rows of any alignment.
struct Bytes {
    const int8_t* data;
    const int8_t* end;  // past the last row's last byte
    size_t stride;
    int rows, cols;
    bool vector;        // rows start on 16 bytes
};

// 16 bytes of a row from column c on, zeros beyond its end.  An unaligned row is
// read in the aligned words that cover it, wherever those lie inside the matrix.
__device__ __forceinline__ uint4 load_bytes(const Bytes& m, const int8_t* row, int c) {
    const int left = m.cols - c;
    if (m.vector && left >= 16) return __ldg(reinterpret_cast<const uint4*>(row + c));
    uint32_t out[4] = {};
    if (left > 0) {
        const int8_t* p = row + c;
        const unsigned shift = reinterpret_cast<uintptr_t>(p) & 3u;
        const int8_t* first = p - shift;
        if (first >= m.data && first + 20 <= m.end) {
            uint32_t w[5];
#pragma unroll
            for (int i = 0; i < 5; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(first) + i);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int keep = left - 4 * i;
                const uint32_t v = __funnelshift_r(w[i], w[i + 1], 8 * shift);
                out[i] = keep >= 4 ? v : keep > 0 ? v & ((1u << (8 * keep)) - 1) : 0u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < left) out[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * (j & 3));
        }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Rows of bytes into rows that start on 16 bytes, for the TMA; bytes up to the
// next multiple of 16 become zeros.
struct RepackArgs {
    Bytes src;
    int8_t* dst;
    size_t dst_stride;
};

__device__ void repack_rows(const RepackArgs& a, unsigned block, unsigned blocks) {
    const int64_t units = (a.src.cols + 15) / 16, n = a.src.rows * units;
    for (int64_t i = static_cast<int64_t>(block) * kThreads + threadIdx.x; i < n; i += static_cast<int64_t>(blocks) * kThreads) {
        const int64_t r = i / units;
        const int c = static_cast<int>(i - r * units) * 16;
        *reinterpret_cast<uint4*>(a.dst + r * a.dst_stride + c) = load_bytes(a.src, a.src.data + r * a.src.stride, c);
    }
}

__global__ void __launch_bounds__(kThreads) repack_kernel(const RepackArgs a) { repack_rows(a, blockIdx.x, gridDim.x); }

// ------------------------------------------------------------------ quantisation
struct QuantizeArgs {
    const void* x;
    const void* x_end;  // past the last row's last element
    size_t x_stride;
    int8_t* q;
    size_t q_stride;
    float* scales;
    int rows, cols;
    int padded_cols;  // columns [cols, padded_cols) of q are zeroed
    bool q_vector;    // 16-byte aligned rows of q, padded_cols a multiple of 16
    unsigned ctas;    // the CTAs after these repack the weights
    RepackArgs weights;
};

constexpr int kGroup = 16;  // columns that a thread takes together: a 16-byte store of q

// Which of the aligned 16-byte units around a row lie inside its matrix; the row's
// values in the others are loaded one by one.
struct RowUnits {
    bool first_out, last_out;
    const uint4* past;  // the units that may be read end here
};

template <typename T>
__device__ __forceinline__ RowUnits row_units(const QuantizeArgs& a, const T* x, int cols) {
    auto down = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15); };
    const uintptr_t past = down(reinterpret_cast<const char*>(x + cols) + 15), end = down(a.x_end);
    return {down(x) < reinterpret_cast<uintptr_t>(a.x), past > end, reinterpret_cast<const uint4*>(min(past, end))};
}

// kGroup values of a row as they are in memory.
template <typename T>
struct Group {
    uint4 raw[kGroup * sizeof(T) / 16];
    __device__ __forceinline__ void load_elements(const T* x, int c, int cols) {
        T* e = reinterpret_cast<T*>(raw);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) e[i] = c + i < cols ? x[c + i] : from_f32<T>(0.0f);
    }
    // A row that starts on 16 bytes.
    __device__ __forceinline__ void load(const T* x, int c, int cols) {
        constexpr int kUnits = kGroup * sizeof(T) / 16;
        if (c + kGroup <= cols) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(x + c) + i);
        } else {
            load_elements(x, c, cols);
        }
    }
    // The same of a row at any alignment: the aligned units that hold the values,
    // shifted into place; units without a value of the row are not read, nor those
    // that stick out of the matrix.  (Loads of single elements took 31 us for 3373
    // rows of 5445 bf16, these 24.)
    __device__ __forceinline__ void load_shifted(const T* x, int c, int cols, const RowUnits& units) {
        constexpr int kUnits = kGroup * sizeof(T) / 16;
        const char* const at = reinterpret_cast<const char*>(x + c);
        const unsigned offset = static_cast<unsigned>(reinterpret_cast<uintptr_t>(at)) & 15;
        const uint4* const from = reinterpret_cast<const uint4*>(at - offset);
        uint32_t w[4 * kUnits + 4];
#pragma unroll
        for (int i = 0; i <= kUnits; ++i) {
            const bool some = c < cols && from + i < units.past && (i > 0 || c > 0 || !units.first_out) && (i < kUnits || offset != 0);
            const uint4 u = some ? __ldcs(from + i) : make_uint4(0, 0, 0, 0);
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
#pragma unroll
        for (int step = 2; step >= 1; step /= 2)
#pragma unroll
            for (int i = 0; i + step < 4 * kUnits + 4; ++i)
                if (offset & (4 * step)) w[i] = w[i + step];
#pragma unroll
        for (int i = 0; i < 4 * kUnits; ++i) {
            const int left = min(cols - c, kGroup) * static_cast<int>(sizeof(T)) - 4 * i;  // bytes of the row from here on, in this group
            const uint32_t word = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (offset & 2) * 8) : w[i];
            reinterpret_cast<uint32_t*>(raw)[i] = left >= 4 ? word : left > 0 ? word & 0xffffu : 0;
        }
    }
    // The values in units that stick out.
    __device__ __forceinline__ void load_rest(const T* x, int c, int cols, const RowUnits& units) {
        const void* const past = x + min(c + kGroup, cols);
        if (c < cols && ((c == 0 && units.first_out) || past > units.past)) load_elements(x, c, cols);
    }
    __device__ __forceinline__ float get(int i) const { return to_f32(reinterpret_cast<const T*>(raw)[i]); }
    // max |x|; NaN becomes +inf
    __device__ __forceinline__ float top() const {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < kGroup; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(t) : "f"(fabsf(get(i))));
        return t == t ? t : INFINITY;
    }
    __device__ __forceinline__ void store(const QuantizeArgs& a, int8_t* q, int c, float factor, bool some) const {
        uint32_t words[kGroup / 4];
#pragma unroll
        for (int w = 0; w < kGroup / 4; ++w) {
            words[w] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                words[w] |= (static_cast<uint32_t>(quantised(get(4 * w + j), factor)) & 0xffu) << (8 * j);
            if (!some) words[w] = 0;
        }
        if (a.q_vector) {
            *reinterpret_cast<uint4*>(q + c) = make_uint4(words[0], words[1], words[2], words[3]);
        } else {
#pragma unroll
            for (int i = 0; i < kGroup; ++i)
                if (c + i < a.padded_cols) q[c + i] = static_cast<int8_t>(words[i >> 2] >> (8 * (i & 3)));
        }
    }
};

// kRowThreads threads for each row, which hold its values in registers between
// the maximum and the rounding: x is read once.  Rows longer than 2 * kGroup *
// kRowThreads (only with kRowThreads == kThreads) read the rest again, from L2.
// 16384 x 4096 bf16: 38 us, 5.2 TB/s, bound by memory and the conversions together
// (61 % of the issue slots); with the values held as f32, 92 registers and 16
// warps on an SM it took 67 us.
template <typename T, int kRowThreads, bool kAligned>
__global__ void __launch_bounds__(kThreads, 4) quantize_kernel(const QuantizeArgs a) {
    constexpr int kHeld = 2, kRowWarps = kRowThreads / 32;
    __shared__ float warp_top[kWarps];
    let_next_start();
    if (blockIdx.x >= a.ctas) {
        repack_rows(a.weights, blockIdx.x - a.ctas, gridDim.x - a.ctas);
        return;
    }
    const int in_row = threadIdx.x % kRowThreads;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / kRowThreads) + threadIdx.x / kRowThreads;
    const bool live = row < a.rows;
    const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
    const int cols = live ? a.cols : 0;
    const RowUnits units = row_units(a, x, cols);
    Group<T> held[kHeld];
    auto load = [&](Group<T>& g, int c) {
        if constexpr (kAligned) g.load(x, c, cols);
        else g.load_shifted(x, c, cols, units);
    };
    auto load_rest = [&](Group<T>& g, int c) {
        if (!kAligned && (units.first_out || units.last_out)) g.load_rest(x, c, cols, units);
    };
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) load(held[j], (in_row + j * kRowThreads) * kGroup);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) load_rest(held[j], (in_row + j * kRowThreads) * kGroup);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) top = fmaxf(top, held[j].top());
    for (int c = (in_row + kHeld * kRowThreads) * kGroup; c < cols; c += kRowThreads * kGroup) {
        Group<T> g;
        load(g, c);
        load_rest(g, c);
        top = fmaxf(top, g.top());
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (kRowWarps > 1) {
        if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
        __syncthreads();
        const int first = (threadIdx.x >> 5) / kRowWarps * kRowWarps;
#pragma unroll
        for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, warp_top[first + w]);
    }
    if (!live) return;
    const bool some = top >= kSmallest && top < INFINITY;
    const float factor = some ? row_factor(top) : 0.0f;
    int8_t* q = a.q + row * a.q_stride;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int c = (in_row + j * kRowThreads) * kGroup;
        if (c < a.padded_cols) held[j].store(a, q, c, factor, some);
    }
    for (int c = (in_row + kHeld * kRowThreads) * kGroup; c < a.padded_cols; c += kRowThreads * kGroup) {
        Group<T> g;
        load(g, c);
        load_rest(g, c);
        g.store(a, q, c, factor, some);
    }
    if (in_row == 0) a.scales[row] = top == INFINITY ? NAN : some ? row_scale(top) : 0.0f;
}

// ------------------------------------------------------------------ few rows
// For one or two rows the weights' bytes are what counts: every warp takes
// output channels one after the other, 16 bytes of a channel for each lane at
// a time, against the rows' 8-bit values in shared memory.  Each CTA quantises
// the rows itself (they are a few KB from L2), so the layer is one launch, and
// the first channel's weights are on their way meanwhile.  One row of 1536 x 2048
// takes 3.8 us, which is the launch and one chain of latencies; two rows of 4096
// x 4096 8.2 us against 9.2 on the tensor cores, four were 16 against 9.
constexpr int kFewRows = 2;
// Shared memory for the rows: what a launch has without asking for more, less the
// kernel's own row maxima.
constexpr size_t kFewRowsBytes = 48 * 1024 - kWarps * kFewRows * sizeof(float);

struct FewRowsArgs {
    ProductArgs p;
    bool quantise;  // the rows are x; otherwise p.q and p.scales
    const void* x;
    size_t x_stride;
    Bytes w;
};

template <typename T, typename Out, int kRows>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const FewRowsArgs a) {
    extern __shared__ uint4 shared_rows[];  // [kRows][pitch] bytes
    __shared__ float tops[kWarps][kRows];
    constexpr int kAhead = 4;
    const ProductArgs& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pitch = (p.k + 15) / 16 * 16;
    int8_t* const rows = reinterpret_cast<int8_t*>(shared_rows);
    int64_t n = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    const int64_t first_end = static_cast<int64_t>(blockIdx.x + 1) * kWarps;
    uint4 ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int c = (i * 32 + lane) * 16;
        ahead[i] = n < p.n ? load_bytes(a.w, p.w + n * p.w_stride, c) : make_uint4(0, 0, 0, 0);
    }
    float scale[kRows];
    if (a.quantise) {
        const T* x = static_cast<const T*>(a.x);
        float top[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            top[r] = 0.0f;
            if (r < p.m)
                for (int c = threadIdx.x; c < p.k; c += kThreads) {
                    const float m = fabsf(to_f32(x[r * a.x_stride + c]));
                    top[r] = fmaxf(top[r], m == m ? m : INFINITY);
                }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], d));
            if (lane == 0) tops[warp][r] = top[r];
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top[r] = fmaxf(top[r], tops[w][r]);
            const bool some = top[r] >= kSmallest && top[r] < INFINITY;
            const float factor = some ? row_factor(top[r]) : 0.0f;
            scale[r] = top[r] == INFINITY ? NAN : some ? row_scale(top[r]) : 0.0f;
            for (int c = threadIdx.x; c < pitch; c += kThreads)
                rows[r * pitch + c] = static_cast<int8_t>(
                    some && r < p.m && c < p.k ? quantised(to_f32(x[r * a.x_stride + c]), factor) : 0);
        }
    } else {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            scale[r] = r < p.m ? p.scales[r] : 0.0f;
            for (int c = threadIdx.x; c < pitch; c += kThreads)
                rows[r * pitch + c] = r < p.m && c < p.k ? p.q[r * p.q_stride + c] : 0;
        }
    }
    __syncthreads();
    for (; n < p.n; n += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int8_t* w = p.w + n * p.w_stride;
        int sum[kRows] = {};
        auto take = [&](const uint4& v, int c) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const int4 q = *reinterpret_cast<const int4*>(rows + r * pitch + c);
                sum[r] = __dp4a(static_cast<int>(v.x), q.x, sum[r]);
                sum[r] = __dp4a(static_cast<int>(v.y), q.y, sum[r]);
                sum[r] = __dp4a(static_cast<int>(v.z), q.z, sum[r]);
                sum[r] = __dp4a(static_cast<int>(v.w), q.w, sum[r]);
            }
        };
        for (int c0 = lane * 16; c0 < p.k; c0 += kAhead * 512) {
            uint4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int c = c0 + i * 512;
                const bool first = n < first_end && c0 == lane * 16;
                v[i] = first ? ahead[i] : load_bytes(a.w, w, c);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (c0 + i * 512 < p.k) take(v[i], c0 + i * 512);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], d);
        if (lane == 0) {
            const float ws = p.w_scales[n], b = p.bias != nullptr ? p.bias[n] : 0.0f;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (r < p.m)
                    static_cast<Out*>(p.out)[r * p.out_stride + n] = from_f32<Out>(int8_result(sum[r], scale[r], ws, b));
        }
    }
}

// ------------------------------------------------------------------ host
size_t padded(size_t n, size_t to) { return (n + to - 1) / to * to; }

unsigned repack_ctas(const BulletOuCudaCppContext* ctx, const RepackArgs& a) {
    const int64_t units = a.src.rows * ((static_cast<int64_t>(a.src.cols) + 15) / 16);
    return static_cast<unsigned>(std::min<int64_t>((units + kThreads - 1) / kThreads, ctx->sm_count * 8));
}

template <typename T, int kRowThreads, bool kAligned>
int launch_quantize(BulletOuCudaCppContext* ctx, QuantizeArgs a) {
    constexpr int kRows = kThreads / kRowThreads;
    a.ctas = static_cast<unsigned>((static_cast<int64_t>(a.rows) + kRows - 1) / kRows);
    const unsigned more = a.weights.src.rows > 0 ? repack_ctas(ctx, a.weights) : 0;
    return launch_kernel(ctx, "int8 quantise launch", quantize_kernel<T, kRowThreads, kAligned>, LaunchShape{dim3(a.ctas + more), kThreads}, a);
}

template <typename T, bool kAligned>
int launch_quantize(BulletOuCudaCppContext* ctx, const QuantizeArgs& a) {
    const int cols = std::max(a.cols, a.padded_cols);
    if (cols <= 32 * 32) return launch_quantize<T, 32, kAligned>(ctx, a);
    if (cols <= 64 * 32) return launch_quantize<T, 64, kAligned>(ctx, a);
    if (cols <= 128 * 32) return launch_quantize<T, 128, kAligned>(ctx, a);
    return launch_quantize<T, 256, kAligned>(ctx, a);
}

// `weights`: rows to repack in the same launch (none: no rows).
int quantize(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix& x, int8_t* q, size_t q_stride, int padded_cols,
             float* scales, const RepackArgs& weights) {
    QuantizeArgs a{};
    a.x = x.data;
    a.x_end = static_cast<const char*>(x.data) + (x.cols > 0 ? (x.rows - 1) * (x.rows > 1 ? x.row_stride : 0) + x.cols : 0) * type_bytes(x.type);
    a.x_stride = x.row_stride;
    a.q = q;
    a.q_stride = q_stride;
    a.scales = scales;
    a.rows = static_cast<int>(x.rows);
    a.cols = static_cast<int>(x.cols);
    a.padded_cols = padded_cols;
    a.q_vector = padded_cols % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && (x.rows <= 1 || q_stride % 16 == 0);
    a.weights = weights;
    if (x.type == BULLETOU_B200_TYPE_F32)
        return rows_aligned(x, 16) ? launch_quantize<float, true>(ctx, a) : launch_quantize<float, false>(ctx, a);
    return rows_aligned(x, 16) ? launch_quantize<__nv_bfloat16, true>(ctx, a) : launch_quantize<__nv_bfloat16, false>(ctx, a);
}

// Whether TMA can read these rows as they are.
bool tma_rows(const void* data, size_t rows, size_t stride) {
    return reinterpret_cast<uintptr_t>(data) % 16 == 0 && (rows <= 1 || stride % 16 == 0);
}

int repack(BulletOuCudaCppContext* ctx, const RepackArgs& a) {
    return launch_kernel(ctx, "int8 repack launch", repack_kernel, LaunchShape{dim3(repack_ctas(ctx, a)), kThreads}, a);
}

Bytes bytes_of(const int8_t* data, size_t stride, int rows, int cols) {
    return {data, data + (rows > 0 ? (rows - 1) * stride + cols : 0), stride, rows, cols, tma_rows(data, rows, stride)};
}

template <typename T, typename Out>
void launch_few_rows(BulletOuCudaCppContext* ctx, const FewRowsArgs& a) {
    const int grid = std::min((a.p.n + kWarps - 1) / kWarps, ctx->sm_count * 4);
    const size_t row = padded(a.p.k, 16);
    if (a.p.m <= 1) few_rows_kernel<T, Out, 1><<<grid, kThreads, row, ctx->stream>>>(a);
    else few_rows_kernel<T, Out, kFewRows><<<grid, kThreads, kFewRows * row, ctx->stream>>>(a);
}

template <typename T>
int few_rows(BulletOuCudaCppContext* ctx, const FewRowsArgs& a, int out_type) {
    if (out_type == BULLETOU_B200_TYPE_F32) launch_few_rows<T, float>(ctx, a);
    else launch_few_rows<T, __nv_bfloat16>(ctx, a);
    return check_launch("int8 few-rows product launch");
}

// The product of `p`, of x's quantised rows where x is given (p.q and p.scales
// are then filled in here).
int product(BulletOuCudaCppContext* ctx, ProductArgs p, const BulletOuB200Matrix* x, int out_type) {
    if (p.m <= kFewRows && kFewRows * padded(p.k, 16) <= kFewRowsBytes) {
        FewRowsArgs a{};
        a.p = p;
        a.w = bytes_of(p.w, p.w_stride, p.n, p.k);
        if (x != nullptr) {
            a.quantise = true;
            a.x = x->data;
            a.x_stride = x->row_stride;
        }
        if (x != nullptr && x->type == BULLETOU_B200_TYPE_BF16) return few_rows<__nv_bfloat16>(ctx, a, out_type);
        return few_rows<float>(ctx, a, out_type);
    }
    const size_t pitch = std::max<size_t>(padded(p.k, 16), 16);
    const bool own_q = x != nullptr || p.k == 0 || !tma_rows(p.q, p.m, p.q_stride);
    const bool own_w = p.k == 0 || !tma_rows(p.w, p.n, p.w_stride);
    const size_t scale_bytes = padded(static_cast<size_t>(p.m) * sizeof(float), 256);
    const size_t q_bytes = own_q ? padded(p.m * pitch, 256) : 0;
    void* scratch = nullptr;
    if (scratch_slot(ctx, kScratchInt8, scale_bytes + q_bytes + (own_w ? p.n * pitch : 0), &scratch, "cudaMalloc int8 rows") != 0)
        return -1;
    float* const scales = static_cast<float*>(scratch);
    int8_t* const q = static_cast<int8_t*>(scratch) + scale_bytes;
    int8_t* const w = q + q_bytes;
    RepackArgs weights{};
    if (own_w) {
        if (p.k > 0) weights = {bytes_of(p.w, p.w_stride, p.n, p.k), w, pitch};
        p.w = w;
        p.w_stride = pitch;
    }
    if (x != nullptr) {
        if (quantize(ctx, *x, q, pitch, static_cast<int>(pitch), scales, weights) != 0) return -1;
        p.scales = scales;
    } else {
        if (weights.src.rows > 0 && repack(ctx, weights) != 0) return -1;
        if (own_q && p.k > 0 && repack(ctx, {bytes_of(p.q, p.q_stride, p.m, p.k), q, pitch}) != 0) return -1;
    }
    if (own_q) {
        p.q = q;
        p.q_stride = pitch;
    }
    // a single row's stride is the caller's and may be anything
    if (p.m == 1) p.q_stride = pitch;
    if (p.n == 1) p.w_stride = pitch;
    return launch_int8_mma(ctx, p, out_type, x != nullptr, weights.src.rows == 0);
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
                    static_cast<float*>(scales->data), RepackArgs{}) != 0
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
    return product(ctx, a, nullptr, out->type) != 0 ? -1 : ok();
}

int bulletou_b200_int8_linear_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* x,
                                     const BulletOuB200Matrix* weights, const BulletOuB200Matrix* weight_scales,
                                     const BulletOuB200Matrix* bias, const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(x, kTypeFloat, "int8 x") != 0 ||
        validate_weights(x, "x", weights, weight_scales, bias, out) != 0)
        return -1;
    ProductArgs a = product_args(*weights, *weight_scales, bias, *out);
    if (a.m == 0 || a.n == 0) return ok();
    return product(ctx, a, x, out->type) != 0 ? -1 : ok();
}

}  // extern "C"
