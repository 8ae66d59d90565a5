// Embedding lookup with scaling, and its gradient by sorted tokens (sm_100a).
//
//   out[n] = scale * table[t_n]            (zeros where t_n is outside the table)
//   table_gradients[v] = scale * sum over n with t_n = v of out_gradients[n]
//
// The gradient sorts the tokens (stable, so each row's entries keep their
// order) and sums the rows of equal tokens in that order: no floating atomics,
// the same bits from call to call.  The sort is a least-significant-digit
// radix sort of (token, position) with tokens outside the table as the largest
// key.
#include <algorithm>

#include "device_matrix.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kTile = 2048;  // keys of one CTA
constexpr int kKeysPerWarp = kTile / kWarps;

// Tokens in row-major order; those outside [0, vocab) become vocab.
struct Tokens {
    const int* data;
    int n;
    int cols;
    size_t row_stride;  // == cols where rows follow one another
    int vocab;
    __device__ __forceinline__ int operator()(int i) const {
        size_t at = i;
        if (row_stride != static_cast<size_t>(cols)) {
            const int r = i / cols;
            at = r * row_stride + (i - r * cols);
        }
        const int t = data[at];
        return t < 0 || t >= vocab ? vocab : t;
    }
};

// ------------------------------------------------------------------ lookup
struct LookupArgs {
    Tokens tokens;
    const void* table;
    void* out;
    int width;
    size_t table_stride, out_stride;
    float scale;
};

template <typename In, typename Out>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const LookupArgs a) {
    const size_t n = static_cast<size_t>(a.tokens.n) * a.width;
    for (size_t i = static_cast<size_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
         i += static_cast<size_t>(gridDim.x) * kThreads) {
        const int row = static_cast<int>(i / a.width);
        const int col = static_cast<int>(i - static_cast<size_t>(row) * a.width);
        const int t = a.tokens(row);
        float v = 0.0f;
        if (t < a.tokens.vocab) v = to_f32(static_cast<const In*>(a.table)[t * a.table_stride + col]) * a.scale;
        static_cast<Out*>(a.out)[row * a.out_stride + col] = from_f32<Out>(v);
    }
}

// ------------------------------------------------------------------ sort
struct SortPass {
    Tokens tokens;           // keys of the first pass
    const int* keys_in;      // null: the tokens themselves, at positions 0..n-1
    const int* positions_in;
    int* keys_out;
    int* positions_out;
    int* counts;             // [bins][tiles], turned into starts inside a bin
    int* totals;             // [bins]
    int n, tiles, shift, bins;
    __device__ __forceinline__ int key(int i) const { return keys_in != nullptr ? keys_in[i] : tokens(i); }
    __device__ __forceinline__ int digit(int k) const { return (k >> shift) & (bins - 1); }
};

__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortPass s) {
    __shared__ int count[kMaxBins];
    for (int b = threadIdx.x; b < s.bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const int first = blockIdx.x * kTile;
    for (int i = first + threadIdx.x; i < min(s.n, first + kTile); i += kThreads) atomicAdd(count + s.digit(s.key(i)), 1);
    __syncthreads();
    for (int b = threadIdx.x; b < s.bins; b += kThreads) s.counts[static_cast<size_t>(b) * s.tiles + blockIdx.x] = count[b];
}

// Exclusive sum of `v` over the block's threads, and the total.
__device__ __forceinline__ int block_exclusive(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    __syncthreads();
    *total = all;
    return before + incl - v;
}

// CTA per bin: where each tile's keys of the bin start inside the bin.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(const SortPass s) {
    __shared__ int warp_sums[kWarps];
    int* counts = s.counts + static_cast<size_t>(blockIdx.x) * s.tiles;
    int run = 0;
    for (int t0 = 0; t0 < s.tiles; t0 += kThreads) {
        const int t = t0 + threadIdx.x;
        int total;
        const int start = block_exclusive(t < s.tiles ? counts[t] : 0, warp_sums, &total);
        if (t < s.tiles) counts[t] = run + start;
        run += total;
    }
    if (threadIdx.x == 0) s.totals[blockIdx.x] = run;
}

// CTA per tile, each warp a run of consecutive keys: a key's place is the start
// of its bin, its tile's start in the bin, the keys of earlier warps and steps,
// and its rank among the equal digits of its warp's step.
__global__ void __launch_bounds__(kThreads) sort_scatter_kernel(const SortPass s) {
    __shared__ int place[kWarps][kMaxBins];
    __shared__ int warp_sums[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kWarps * kMaxBins; i += kThreads) place[0][i] = 0;
    __syncthreads();
    const int first = blockIdx.x * kTile + warp * kKeysPerWarp;
    const int end = min(s.n, first + kKeysPerWarp);
    for (int i = first + lane; i < end; i += 32) atomicAdd(&place[warp][s.digit(s.key(i))], 1);
    __syncthreads();
    int run = 0;
    for (int b0 = 0; b0 < s.bins; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int total;
        int at = run + block_exclusive(b < s.bins ? s.totals[b] : 0, warp_sums, &total);
        run += total;
        if (b < s.bins) {
            at += s.counts[static_cast<size_t>(b) * s.tiles + blockIdx.x];
            for (int w = 0; w < kWarps; ++w) {
                const int c = place[w][b];
                place[w][b] = at;
                at += c;
            }
        }
    }
    __syncthreads();
    for (int i0 = first; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const unsigned active = __ballot_sync(0xffffffffu, i < end);
        if (i < end) {
            const int k = s.key(i);
            const int d = s.digit(k);
            const unsigned peers = __match_any_sync(active, d);
            const int start = place[warp][d];
            const int at = start + __popc(peers & ((1u << lane) - 1));
            s.keys_out[at] = k;
            s.positions_out[at] = s.positions_in != nullptr ? s.positions_in[i] : i;
            __syncwarp(active);  // every lane has read `start`
            if (lane == 31 - __clz(peers)) place[warp][d] = start + __popc(peers);
        }
        __syncwarp();
    }
}

// ------------------------------------------------------------------ gradient
struct GradientArgs {
    const int* keys;       // sorted
    const int* positions;
    int n;
    const void* grad;
    void* out;
    int vocab, width;
    size_t grad_stride, out_stride;
    float scale;
};

// First place in the sorted keys whose key is not below `v`.
__device__ __forceinline__ int lower_bound(const int* keys, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// CTA per table row: its entries summed in order, a thread per column.
template <typename In, typename Out>
__global__ void __launch_bounds__(kThreads) gradient_kernel(const GradientArgs a) {
    __shared__ int range[2];
    const int v = blockIdx.x;
    if (threadIdx.x < 2) range[threadIdx.x] = lower_bound(a.keys, a.n, v + threadIdx.x);
    __syncthreads();
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
        float sum = 0.0f;
        for (int i = range[0]; i < range[1]; ++i)
            sum += to_f32(static_cast<const In*>(a.grad)[a.positions[i] * a.grad_stride + c]);
        static_cast<Out*>(a.out)[v * a.out_stride + c] = from_f32<Out>(sum * a.scale);
    }
}

Tokens tokens_of(const BulletOuB200Matrix& m, size_t vocab) {
    Tokens t{};
    t.data = static_cast<const int*>(m.data);
    t.n = static_cast<int>(m.rows * m.cols);
    t.cols = static_cast<int>(m.cols);
    t.row_stride = is_flat(m) ? m.cols : m.row_stride;
    t.vocab = static_cast<int>(vocab);
    return t;
}

int validate_tokens(const BulletOuB200Matrix* tokens, const char* name) {
    if (validate_matrix(tokens, kTypeI32, name) != 0) return -1;
    if (tokens->rows * tokens->cols >= static_cast<size_t>(INT32_MAX) - kTile)
        return fail_messagef("%s: too many tokens (%zu)", name, tokens->rows * tokens->cols);
    return 0;
}

// Sorts the tokens into context scratch.
int sort_tokens(BulletOuCudaCppContext* ctx, const Tokens& tokens, const int** keys, const int** positions) {
    const int n = tokens.n;
    const int tiles = (n + kTile - 1) / kTile;
    int bits = 1;
    while (static_cast<int64_t>(tokens.vocab) >> bits != 0) ++bits;
    const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    const int digit_bits = (bits + passes - 1) / passes;
    const int bins = 1 << digit_bits;
    const size_t row = (static_cast<size_t>(n) + 63) / 64 * 64;
    const size_t counts = static_cast<size_t>(bins) * tiles;
    void* p = nullptr;
    if (scratch_slot(ctx, kScratchEmbedding, (4 * row + counts + kMaxBins) * sizeof(int), &p,
                     "cudaMalloc embedding sort") != 0)
        return -1;
    int* const base = static_cast<int*>(p);
    SortPass s{};
    s.tokens = tokens;
    s.n = n;
    s.tiles = tiles;
    s.bins = bins;
    s.totals = base + 4 * row;
    s.counts = s.totals + kMaxBins;
    for (int pass = 0; pass < passes; ++pass) {
        s.shift = pass * digit_bits;
        s.keys_out = base + (pass & 1) * 2 * row;
        s.positions_out = s.keys_out + row;
        sort_count_kernel<<<tiles, kThreads, 0, ctx->stream>>>(s);
        sort_scan_kernel<<<bins, kThreads, 0, ctx->stream>>>(s);
        sort_scatter_kernel<<<tiles, kThreads, 0, ctx->stream>>>(s);
        s.keys_in = s.keys_out;
        s.positions_in = s.positions_out;
    }
    *keys = s.keys_in;
    *positions = s.positions_in;
    return check_launch("embedding sort launch");
}

}  // namespace
}  // namespace bou

using namespace bou;

extern "C" {

int bulletou_b200_embedding_forward_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* table,
                                           const BulletOuB200Matrix* tokens, float scale,
                                           const BulletOuB200Matrix* out) {
    if (set_device(ctx) != 0 || validate_matrix(table, kTypeFloat, "embedding table") != 0 ||
        validate_tokens(tokens, "embedding tokens") != 0 ||
        validate_matrix(out, kTypeFloat, tokens->rows * tokens->cols, table->cols, "embedding out") != 0 ||
        validate_disjoint(out, "embedding out", table, "the table") != 0 ||
        validate_disjoint(out, "embedding out", tokens, "the tokens") != 0)
        return -1;
    LookupArgs a{};
    a.tokens = tokens_of(*tokens, table->rows);
    if (a.tokens.n == 0 || table->cols == 0) return ok();
    a.table = table->data;
    a.out = out->data;
    a.width = static_cast<int>(table->cols);
    a.table_stride = table->row_stride;
    a.out_stride = out->row_stride;
    a.scale = scale;
    const size_t blocks = (static_cast<size_t>(a.tokens.n) * a.width + kThreads - 1) / kThreads;
    const int grid = static_cast<int>(std::min<size_t>(blocks, static_cast<size_t>(ctx->sm_count) * 8));
    const bool in16 = table->type == BULLETOU_B200_TYPE_BF16, out16 = out->type == BULLETOU_B200_TYPE_BF16;
    using B = __nv_bfloat16;
    if (in16 && out16) lookup_kernel<B, B><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (in16) lookup_kernel<B, float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else if (out16) lookup_kernel<float, B><<<grid, kThreads, 0, ctx->stream>>>(a);
    else lookup_kernel<float, float><<<grid, kThreads, 0, ctx->stream>>>(a);
    return check_launch("embedding lookup launch") != 0 ? -1 : ok();
}

int bulletou_b200_embedding_backward_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* tokens,
                                            const BulletOuB200Matrix* out_gradients, float scale,
                                            const BulletOuB200Matrix* table_gradients) {
    if (set_device(ctx) != 0 || validate_tokens(tokens, "embedding tokens") != 0 ||
        validate_matrix(table_gradients, kTypeFloat, "embedding table gradients") != 0 ||
        validate_matrix(out_gradients, kTypeFloat, tokens->rows * tokens->cols, table_gradients->cols,
                        "embedding out gradients") != 0 ||
        validate_disjoint(table_gradients, "embedding table gradients", out_gradients, "the out gradients") != 0 ||
        validate_disjoint(table_gradients, "embedding table gradients", tokens, "the tokens") != 0)
        return -1;
    if (table_gradients->rows == 0 || table_gradients->cols == 0) return ok();
    GradientArgs a{};
    const Tokens t = tokens_of(*tokens, table_gradients->rows);
    a.n = t.n;
    if (t.n > 0 && sort_tokens(ctx, t, &a.keys, &a.positions) != 0) return -1;
    a.grad = out_gradients->data;
    a.out = table_gradients->data;
    a.vocab = t.vocab;
    a.width = static_cast<int>(table_gradients->cols);
    a.grad_stride = out_gradients->row_stride;
    a.out_stride = table_gradients->row_stride;
    a.scale = scale;
    const bool in16 = out_gradients->type == BULLETOU_B200_TYPE_BF16;
    const bool out16 = table_gradients->type == BULLETOU_B200_TYPE_BF16;
    using B = __nv_bfloat16;
    if (in16 && out16) gradient_kernel<B, B><<<a.vocab, kThreads, 0, ctx->stream>>>(a);
    else if (in16) gradient_kernel<B, float><<<a.vocab, kThreads, 0, ctx->stream>>>(a);
    else if (out16) gradient_kernel<float, B><<<a.vocab, kThreads, 0, ctx->stream>>>(a);
    else gradient_kernel<float, float><<<a.vocab, kThreads, 0, ctx->stream>>>(a);
    return check_launch("embedding gradient launch") != 0 ? -1 : ok();
}

}  // extern "C"
