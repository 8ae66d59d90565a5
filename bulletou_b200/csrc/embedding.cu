// Embedding lookup with scaling, and its gradient by sorted tokens (sm_100a).
//
//   out[n] = scale * table[t_n]            (zeros where t_n is outside the table)
//   table_gradients[v] = scale * sum over n with t_n = v of out_gradients[n]
//
// Both are bound by the rows' bytes.  The lookup is one pass with several rows
// in flight for each warp.  The gradient sorts the tokens (stable, so each
// row's entries keep their order) and then sums runs of equal tokens in that
// order: no floating atomics, the same bits from call to call, every row of
// out_gradients read once and every row of the table written once.
#include <algorithm>
#include <climits>
#include <cmath>
#include <utility>

#include "device_matrix.cuh"
#include "token_launch.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kLookupCtas = 5;  // CTAs on an SM

// Tokens in row-major order; those outside [0, vocab) become vocab.
struct Tokens {
    const int* data;
    int n;
    int cols;
    size_t row_stride;  // == cols where rows follow one another
    int vocab;
    __device__ __forceinline__ int checked(int t) const {
        return static_cast<unsigned>(t) < static_cast<unsigned>(vocab) ? t : vocab;
    }
    __device__ __forceinline__ int operator()(int i) const {
        size_t at = i;
        if (row_stride != static_cast<size_t>(cols)) {
            const int r = i / cols;
            at = r * row_stride + (i - r * cols);
        }
        return checked(data[at]);
    }
};

// kUnit elements that are loaded or stored together, as they are in memory: 16
// bytes of the narrower type where the rows allow it, else one element.
template <typename T, int kUnit>
struct Raw {
    static constexpr int kWords = kUnit == 1 ? 1 : kUnit * static_cast<int>(sizeof(T)) / 4;  // 1, 2, 4 or 8
    uint32_t w[kWords];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kUnit == 1) {
            if constexpr (sizeof(T) == 2) w[0] = *reinterpret_cast<const unsigned short*>(p);  // the whole word, so that none is merged
            else w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kWords == 1) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kWords == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            w[0] = u.x, w[1] = u.y;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 u = *(reinterpret_cast<const uint4*>(p) + i / 4);
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kUnit == 1) {
            *p = *reinterpret_cast<const T*>(w);
        } else if constexpr (kWords == 1) {
            __stcs(reinterpret_cast<uint32_t*>(p), w[0]);
        } else if constexpr (kWords == 2) {
            __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                __stcs(reinterpret_cast<uint4*>(p) + i / 4, make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
        }
    }
    __device__ __forceinline__ float get(int j) const { return to_f32(reinterpret_cast<const T*>(w)[j]); }
    __device__ __forceinline__ void set(int j, float v) { reinterpret_cast<T*>(w)[j] = from_f32<T>(v); }
};
// The vector unit of a pair of types: 8 bf16 or 4 f32 fill 16 bytes.
template <typename A, typename B>
constexpr int kVectorUnit = sizeof(A) == 2 && sizeof(B) == 2 ? 8 : 4;

// ------------------------------------------------------------------ lookup
struct LookupArgs {
    Tokens tokens;
    const void* table;
    void* out;
    int width;
    size_t table_stride, out_stride;
    float scale;
};

// A group of 2^k lanes, enough for a row's units, takes `span` neighbouring rows
// (at most a row for each lane): each lane fetches one row's token, and the
// rows' units are then loaded kRows at a time, all in flight together.  The
// stores stream past L2, which keeps the table.
//
// Bound by the stores: 655360 rows of 256 bf16 take 71 to 74 us, 5.2 TB/s of which
// 4.6 are written (torch's fill of that output alone takes 89 us).  With rows
// held as f32, 70 registers and 24 warps on an SM it took 109 us.  Units of one or
// two elements are bound by latency: rows of more than 32 of them have kCols
// units of each row in flight in a lane, 155642 rows of 257 f32 46 us instead of
// 66, 600000 of 63 bf16 37 instead of 55.  Aligned 16-byte blocks shifted into
// place took 79 us there: all lanes go through the rows' ends element by element.
//
// kAnyScale: a scale that is not finite, which would not leave a padded token's
// zeros as they are (a select of every row's scale cost finite ones up to 7 %).
template <typename In, typename Out, int kUnit, int kCols, bool kAnyScale = false>
__global__ void __launch_bounds__(kThreads, kLookupCtas) lookup_kernel(const LookupArgs a, int any_group, int span) {
    constexpr int kRows = 4;
    const int group = kCols > 1 ? 32 : any_group;  // with a group known only at run time the columns' offsets cost 100 bytes of spills
    const int lane = threadIdx.x & (group - 1);
    // blockIdx.y cuts the columns
    const int share = (a.width / kUnit + gridDim.y - 1) / gridDim.y;
    const int unit0 = blockIdx.y * share, units = min(a.width / kUnit, unit0 + share);
    const int64_t groups = static_cast<int64_t>(gridDim.x) * (kThreads / group);
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / group;
    // the lanes of a warp stay together for the shuffles: a group past the end has no rows
    for (int64_t r0 = first * span; __any_sync(0xffffffffu, r0 < a.tokens.n); r0 += groups * span) {
        const int rows = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(span), a.tokens.n - r0)));
        const int own = lane < rows ? a.tokens(static_cast<int>(r0) + lane) : a.tokens.vocab;
        const In* const table = static_cast<const In*>(a.table);
        Out* const out = static_cast<Out*>(a.out) + r0 * a.out_stride;
        for (int i0 = 0; i0 < span; i0 += kRows) {
            int token[kRows];
#pragma unroll
            for (int i = 0; i < kRows; ++i) token[i] = __shfl_sync(0xffffffffu, own, i0 + i, group);
            for (int u = unit0 + lane; u < units; u += group * kCols) {
                Raw<In, kUnit> v[kRows][kCols];
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    const In* const row = table + token[i] * a.table_stride + u * kUnit;
#pragma unroll
                    for (int k = 0; k < kCols; ++k) {
                        if (i0 + i < rows && token[i] < a.tokens.vocab && (k == 0 || u + k * group < units)) v[i][k].load(row + k * group * kUnit);
                        else v[i][k].clear();
                    }
                }
#pragma unroll
                for (int i = 0; i < kRows; ++i) {
                    if (i0 + i >= rows) break;
                    const float scale = kAnyScale && token[i] >= a.tokens.vocab ? 0.0f : a.scale;
                    Out* const row = out + (i0 + i) * a.out_stride + u * kUnit;
#pragma unroll
                    for (int k = 0; k < kCols; ++k) {
                        Raw<Out, kUnit> y;
#pragma unroll
                        for (int j = 0; j < kUnit; ++j) y.set(j, v[i][k].get(j) * scale);
                        if (k == 0 || u + k * group < units) y.store(row + k * group * kUnit);
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------ sort
// Least-significant-digit radix sort of (token, position), tokens outside the
// table as the largest key.  Digits of up to 11 bits: fewer passes save three
// launches each, which is what a sort of 10^5 tokens costs, and 2048 counters
// for each of 8 warps still fit the shared memory twice.  1310720 tokens of a
// 17-bit table (two passes) take about 45 us, 68438 of an 11-bit one about 15:
// launches, and scattered 8-byte stores.
constexpr int kMaxDigitBits = 11;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kMaxTile = 2048;

struct SortPass {
    Tokens tokens;           // keys of the first pass
    const int2* in;          // (token, position); null: the tokens themselves, at positions 0..n-1
    int2* out;
    int* counts;             // [bins][tiles], turned into starts inside a bin
    int* totals;             // [bins]
    int n, tiles, shift, bins;
    __device__ __forceinline__ int2 entry(int i) const { return in != nullptr ? in[i] : make_int2(tokens(i), i); }
    __device__ __forceinline__ int digit(int k) const { return (k >> shift) & (bins - 1); }
};

template <int kSteps>
__global__ void __launch_bounds__(kThreads) sort_count_kernel(const SortPass s) {
    __shared__ int count[kMaxBins];
    let_next_start();
    for (int b = threadIdx.x; b < s.bins; b += kThreads) count[b] = 0;
    __syncthreads();
    wait_for_previous();
    const int first = blockIdx.x * (kSteps * kThreads) + threadIdx.x;
    int key[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) key[j] = first + j * kThreads < s.n ? s.entry(first + j * kThreads).x : -1;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
        if (key[j] >= 0) atomicAdd(count + s.digit(key[j]), 1);
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

// CTA per bin: where each tile's keys of the bin start inside the bin.  It does
// not let the scatter start early: that cost 8 us of 39 for 68438 tokens.
__global__ void __launch_bounds__(kThreads) sort_scan_kernel(const SortPass s) {
    __shared__ int warp_sums[kWarps];
    wait_for_previous();
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

// CTA per tile, each warp a run of consecutive entries: an entry's place is the
// start of its bin, its tile's start in the bin, the entries of earlier warps,
// and its rank among the equal digits of its warp.
template <int kSteps, int kBinsOfThread>
__global__ void __launch_bounds__(kThreads, kBinsOfThread <= 2 ? 5 : 2) sort_scatter_kernel(const SortPass s) {
    extern __shared__ int places[];  // [kWarps][bins]
    __shared__ int warp_sums[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* const place = places + warp * s.bins;
    let_next_start();
    const int bin0 = threadIdx.x * kBinsOfThread;
    for (int i = threadIdx.x; i < kWarps * s.bins; i += kThreads) places[i] = 0;
    __syncthreads();
    wait_for_previous();
    const int first = blockIdx.x * (kSteps * kThreads) + warp * (kSteps * 32) + lane;
    int2 entry[kSteps];
    int rank[kSteps];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) entry[j] = first + j * 32 < s.n ? s.entry(first + j * 32) : make_int2(-1, 0);
    int total[kBinsOfThread], start[kBinsOfThread];
#pragma unroll
    for (int i = 0; i < kBinsOfThread; ++i) {
        const bool in = bin0 + i < s.bins;
        total[i] = in ? s.totals[bin0 + i] : 0;
        start[i] = in ? s.counts[static_cast<size_t>(bin0 + i) * s.tiles + blockIdx.x] : 0;
    }
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
        // the lanes with this lane's digit; those past the last entry go by themselves
        const bool live = entry[j].x >= 0;
        const int d = live ? s.digit(entry[j].x) : 0;
        unsigned peers = __ballot_sync(0xffffffffu, live);
        peers = live ? peers : ~peers;
#pragma unroll
        for (int bit = 1; bit < kThreads * kBinsOfThread; bit <<= 1) {
            if (bit >= s.bins) break;
            const unsigned set = __ballot_sync(0xffffffffu, d & bit);
            peers &= d & bit ? set : ~set;
        }
        const int before = live ? place[d] : 0;
        __syncwarp();  // every lane has read it
        rank[j] = before + __popc(peers & ((1u << lane) - 1));
        if (live && lane == 31 - __clz(peers)) place[d] = before + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kBinsOfThread; ++i) sum += total[i];
    int all;
    int at = block_exclusive(sum, warp_sums, &all);
#pragma unroll
    for (int i = 0; i < kBinsOfThread; ++i) {
        if (bin0 + i < s.bins) {
            int next = at + start[i];
            for (int w = 0; w < kWarps; ++w) {
                const int c = places[w * s.bins + bin0 + i];
                places[w * s.bins + bin0 + i] = next;
                next += c;
            }
        }
        at += total[i];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
        if (entry[j].x >= 0) s.out[place[s.digit(entry[j].x)] + rank[j]] = entry[j];
}

// Few tokens are ranked instead, in one launch: a token's place is the number of
// tokens that are smaller, or equal and earlier.  A CTA ranks kRankTokens of
// them, kRankParts threads for each, against all n in shared memory.  The gradient
// of 4096 tokens x 64 takes 18 us with it and 23 with the radix sort, of 8192 25
// and 24, of 24 tokens 7 and 16.
constexpr int kRankMost = 4096;
constexpr int kRankTokens = 64;
constexpr int kRankParts = kThreads / kRankTokens;

__global__ void __launch_bounds__(kThreads) rank_tokens_kernel(const Tokens tokens, int2* out) {
    extern __shared__ int4 shared_tokens[];
    __shared__ int ranks[kRankParts][kRankTokens];
    int* const all = reinterpret_cast<int*>(shared_tokens);
    const int n = tokens.n, padded = (n + 3) / 4 * 4;
    let_next_start();
    for (int i = threadIdx.x; i < padded; i += kThreads) all[i] = i < n ? tokens(i) : INT_MAX;
    __syncthreads();
    const int slot = threadIdx.x % kRankTokens, part = threadIdx.x / kRankTokens;
    const int first = blockIdx.x * kRankTokens, i = first + slot;
    const int mine = i < n ? all[i] : INT_MAX;
    // four tokens at a time; those before this CTA's come first among equals, those after it do not
    int rank = 0;
    const int quads = padded / 4, q0 = first / 4, q1 = min(quads, q0 + kRankTokens / 4);
    for (int q = part; q < q0; q += kRankParts) {
        const int4 t = shared_tokens[q];
        rank += (t.x <= mine) + (t.y <= mine) + (t.z <= mine) + (t.w <= mine);
    }
    for (int q = q0 + part; q < q1; q += kRankParts)
        for (int j = 0; j < 4; ++j) {
            const int other = 4 * q + j;
            rank += all[other] < mine || (all[other] == mine && other < i);
        }
    for (int q = q1 + part; q < quads; q += kRankParts) {
        const int4 t = shared_tokens[q];
        rank += (t.x < mine) + (t.y < mine) + (t.z < mine) + (t.w < mine);
    }
    ranks[part][slot] = rank;
    __syncthreads();
    if (part == 0 && i < n) {
        for (int p = 1; p < kRankParts; ++p) rank += ranks[p][slot];
        out[rank] = make_int2(mine, i);
    }
}

// ------------------------------------------------------------------ gradient
// The sorted entries are cut into chunks of equal length, so that a token that
// half of the entries name costs no more than the others.  A group of lanes
// sums its chunk's runs of equal tokens in order.  A run inside the chunk is a
// row's gradient and is written; a run that goes on beyond the chunk leaves a
// partial row, and joined_rows_kernel adds those up in the order of the chunks.
//
// Bound by reading the gradients once: 1310720 rows of 256 f32 take 225 us, 6.3
// TB/s (97 % of a copy), with 4 rows in flight for each of 24 warps on an SM; 8
// rows in flight needed 142 registers, left 8 warps and took 309 us.  Rows of an
// odd width go one element at a time: 68438 of 257 f32 in 16 us, 4.4 TB/s.
struct GradientArgs {
    const int2* entries;   // (token, position), sorted by token
    int n, chunk, chunks;
    const void* grad;
    void* out;
    int vocab, width;
    size_t grad_stride, out_stride;
    float scale;
    // partial rows, part_stride floats apart (whole 16 bytes), one for each chunk:
    float* heads;          // the chunk's first run, begun before it
    float* tails;          // the run that begins in the chunk and goes on after it
    size_t part_stride;
    int row_blocks;        // CTAs that write the rows no token names
};

constexpr int kEmptyRows = 128;  // table rows of one such CTA

// First place in the sorted entries whose token is not below `v`.
__device__ __forceinline__ int lower_bound(const int2* entries, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (entries[mid].x < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <typename Out, int kUnit>
__device__ void write_empty_rows(const GradientArgs& a, int block) {
    __shared__ int empty[kEmptyRows];
    const int64_t v0 = static_cast<int64_t>(block) * kEmptyRows;
    if (threadIdx.x < kEmptyRows) {
        const int64_t v = v0 + threadIdx.x;
        bool none = false;
        if (v < a.vocab) {
            const int at = lower_bound(a.entries, a.n, static_cast<int>(v));
            none = at == a.n || a.entries[at].x != v;
        }
        empty[threadIdx.x] = none;
    }
    __syncthreads();
    Raw<Out, kUnit> zeros;
    zeros.clear();
    for (int r = threadIdx.x >> 5; r < kEmptyRows; r += kWarps) {
        if (!empty[r]) continue;
        Out* out = static_cast<Out*>(a.out) + (v0 + r) * a.out_stride;
        for (int u = threadIdx.x & 31; u < a.width / kUnit; u += 32) zeros.store(out + u * kUnit);
    }
}

// kLanes lanes hold kUnits units of a row each; blockIdx.y cuts wider rows.
template <typename In, typename Out, int kUnit, int kLanes, int kUnits>
__global__ void __launch_bounds__(kThreads, 3) gradient_kernel(const GradientArgs a) {
    constexpr int kBatch = kUnit * kUnits > 4 ? 4 : 8;  // rows in flight
    let_next_start();
    wait_for_previous();
    if (static_cast<int>(blockIdx.x) < a.row_blocks) {
        if (blockIdx.y == 0) write_empty_rows<Out, kUnit>(a, blockIdx.x);
        return;
    }
    const int c = (blockIdx.x - a.row_blocks) * (kThreads / kLanes) + threadIdx.x / kLanes;
    if (c >= a.chunks) return;
    const int lane = threadIdx.x & (kLanes - 1);
    const int units = a.width / kUnit;
    const int u0 = blockIdx.y * kLanes * kUnits + lane;
    const int begin = c * a.chunk, end = min(a.n, begin + a.chunk);
    const int before = begin > 0 ? a.entries[begin - 1].x : -1, after = end < a.n ? a.entries[end].x : -1;
    float sum[kUnits][kUnit] = {};
    int current = a.entries[begin].x;
    bool from_before = current == before;
    auto flush = [&](bool goes_on) {
        if (current < a.vocab) {
            float* part = from_before ? a.heads : goes_on ? a.tails : nullptr;
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                const int u = u0 + k * kLanes;
                if (u >= units) continue;
                if (part != nullptr) {
                    Raw<float, kUnit> v;
#pragma unroll
                    for (int j = 0; j < kUnit; ++j) v.set(j, sum[k][j]);
                    v.store(part + c * a.part_stride + u * kUnit);
                } else {
                    Raw<Out, kUnit> v;
#pragma unroll
                    for (int j = 0; j < kUnit; ++j) v.set(j, sum[k][j] * a.scale);
                    v.store(static_cast<Out*>(a.out) + current * a.out_stride + u * kUnit);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) sum[k][j] = 0.0f;
    };
    int2 entry[kBatch];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) entry[b] = i0 + b < end ? a.entries[i0 + b] : make_int2(a.vocab, 0);
    };
    fetch(begin);
    for (int i0 = begin; i0 < end; i0 += kBatch) {
        Raw<In, kUnit> v[kBatch][kUnits];
        int k_now[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            k_now[b] = entry[b].x;
            const In* row = static_cast<const In*>(a.grad) + entry[b].y * a.grad_stride;
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                const int u = u0 + k * kLanes;
                if (entry[b].x < a.vocab && u < units) v[b][k].load(row + u * kUnit);
                else v[b][k].clear();
            }
        }
        fetch(i0 + kBatch);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + b >= end) break;
            if (k_now[b] != current) {
                flush(false);
                current = k_now[b];
                from_before = false;
            }
#pragma unroll
            for (int k = 0; k < kUnits; ++k)
#pragma unroll
                for (int j = 0; j < kUnit; ++j) sum[k][j] += v[b][k].get(j);
        }
    }
    flush(current == after);
}

// CTA for kWarps chunks: the rows whose run begins in a chunk and goes on after
// it.  Runs over up to kShortRun more chunks take a warp each; longer ones are
// shared by strands of the CTA's lanes, each a run of consecutive chunks, and
// joined in a fixed order.  A lane takes eight columns at a time, two 16-byte loads of every
// partial row.  Bound by latency: the run's end is searched 32 chunks at a time
// (a binary search of 20 steps made it 37 us for 10240 chunks of 256 columns, of
// which the longest run covers 245; now 15).
template <typename Out, bool kVector>
__global__ void __launch_bounds__(kThreads, 4) joined_rows_kernel(const GradientArgs a) {
    constexpr int kShortRun = 8, kQuads = 2, kBlock = 128 * kQuads;
    __shared__ int first_key[kWarps], more[kWarps];  // of each chunk's tail run: its row, the chunks after it
    __shared__ float4 part[kWarps][32 * kQuads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    wait_for_previous();
    const int c0 = blockIdx.x * kWarps;
    {
        const int c = c0 + warp;
        int row = -1, count = 0;
        if (c + 1 < a.chunks) {
            const int begin = c * a.chunk, last = begin + a.chunk - 1;
            const int k = a.entries[last].x, next = a.entries[last + 1].x, own = a.entries[begin].x;
            const int before = begin > 0 ? a.entries[begin - 1].x : -1;
            if (k < a.vocab && next == k && !(own == k && before == k)) {
                row = k;
                // Chunks [c + 1, c + 1 + count) begin with the row; the lanes ask 32 chunks at a
                // time, ever closer to the last of them.
                int lo = c + 1, hi = a.chunks;  // chunk lo begins with it, chunk hi does not (or is past the end)
                int stride = 1;
                while (hi - lo > 1) {
                    const int at = lo + (lane + 1) * stride;
                    const bool same = at < hi && a.entries[static_cast<int64_t>(at) * a.chunk].x == k;
                    const int m = __popc(__ballot_sync(0xffffffffu, same));
                    if (m < 32) hi = static_cast<int>(min(static_cast<int64_t>(hi), lo + static_cast<int64_t>(m + 1) * stride));
                    lo += m * stride;
                    stride = (hi - lo + 31) / 32;
                }
                count = lo - c;
            }
        }
        if (lane == 0) {
            first_key[warp] = row;
            more[warp] = count;
        }
    }
    __syncthreads();
    auto add = [](float4& s, const float4& v) { s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w; };
    auto add_heads = [&](int first, int count, int column, float4* s) {
        const float* row = a.heads + first * a.part_stride + column;
#pragma unroll 4
        for (int i = 0; i < count; ++i, row += a.part_stride)
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
                if (column + 128 * j < a.width) add(s[j], *reinterpret_cast<const float4*>(row + 128 * j));
    };
    auto finish = [&](int c, int key, int first_column, float4* s) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j) {
            const int column = first_column + 128 * j;
            if (column >= a.width) continue;
            add(s[j], *reinterpret_cast<const float4*>(a.tails + c * a.part_stride + column));
            const float v[4] = {s[j].x, s[j].y, s[j].z, s[j].w};
            Out* out = static_cast<Out*>(a.out) + key * a.out_stride + column;
            if constexpr (kVector) {
                Raw<Out, 4> y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y.set(i, v[i] * a.scale);
                y.store(out);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (column + i < a.width) out[i] = from_f32<Out>(v[i] * a.scale);
            }
        }
    };
    if (first_key[warp] >= 0 && more[warp] <= kShortRun)
        for (int base = 0; base < a.width; base += kBlock) {
            float4 s[kQuads] = {};
            add_heads(c0 + warp + 1, more[warp], base + lane * 4, s);
            finish(c0 + warp, first_key[warp], base + lane * 4, s);
        }
    for (int w = 0; w < kWarps; ++w) {
        if (first_key[w] < 0 || more[w] <= kShortRun) continue;
        for (int base = 0; base < a.width; base += kBlock) {
            // `side` lanes hold a row's columns, so narrow rows have more strands
            int side = 1;
            while (side < 32 && side * 4 < a.width - base) side *= 2;
            const int strands = kThreads / side, strand = threadIdx.x / side;
            const int share = (more[w] + strands - 1) / strands;
            const int first = min(more[w], strand * share), count = min(more[w], first + share) - first;
            float4 s[kQuads] = {};
            add_heads(c0 + w + 1 + first, count, base + (lane & (side - 1)) * 4, s);
            for (int d = side; d < 32; d *= 2)
#pragma unroll
                for (int j = 0; j < kQuads; ++j)
                    add(s[j], make_float4(__shfl_down_sync(0xffffffffu, s[j].x, d), __shfl_down_sync(0xffffffffu, s[j].y, d),
                                          __shfl_down_sync(0xffffffffu, s[j].z, d), __shfl_down_sync(0xffffffffu, s[j].w, d)));
#pragma unroll
            for (int j = 0; j < kQuads; ++j) part[warp][lane + 32 * j] = s[j];
            __syncthreads();
            if (warp == 0 && lane < side) {
#pragma unroll
                for (int j = 0; j < kQuads; ++j) {
                    s[j] = part[0][lane + 32 * j];
                    for (int x = 1; x < kWarps; ++x) add(s[j], part[x][lane + 32 * j]);
                }
                finish(c0 + w, first_key[w], base + lane * 4, s);
            }
            __syncthreads();
        }
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
    if (tokens->rows * tokens->cols >= static_cast<size_t>(INT32_MAX) - kMaxTile)
        return fail_messagef("%s: too many tokens (%zu)", name, tokens->rows * tokens->cols);
    return 0;
}

// How the sort's and the gradient's scratch is laid out.
struct GradientPlan {
    int tile, tiles, passes, digit_bits;
    int lanes, units, unit;   // shape of gradient_kernel
    int chunk, chunks;
    size_t row, counts, width;
    size_t words() const { return 4 * row + kMaxBins + counts + 2 * static_cast<size_t>(chunks) * width; }
};

GradientPlan plan_gradient(const BulletOuCudaCppContext* ctx, int n, int vocab, int width, int vector_unit, bool vector) {
    GradientPlan p{};
    int bits = 1;
    while (static_cast<int64_t>(vocab) >> bits != 0) ++bits;
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.digit_bits = (bits + p.passes - 1) / p.passes;
    // a CTA for every SM while there are tokens enough
    p.tile = n > kMaxTile / 2 * ctx->sm_count ? kMaxTile : n > kMaxTile / 4 * ctx->sm_count ? kMaxTile / 2 : kMaxTile / 4;
    p.tiles = (n + p.tile - 1) / p.tile;
    p.row = (static_cast<size_t>(n) + 63) / 64 * 64;
    p.counts = ((static_cast<size_t>(1) << p.digit_bits) * p.tiles + 63) / 64 * 64;
    p.width = (static_cast<size_t>(width) + 3) / 4 * 4;  // partial rows in whole units
    p.unit = vector ? vector_unit : 1;
    const int units = width / p.unit;
    p.lanes = units <= 4 ? 4 : units <= 8 ? 8 : units <= 16 ? 16 : 32;
    // up to 8 values for each lane (5 single ones), so that 4 rows in flight fit
    // the registers; a wider row is cut into equal parts
    const int most = p.unit == 1 ? 5 : 8 / p.unit;
    const int parts = (units + p.lanes * most - 1) / (p.lanes * most);
    p.units = (units + p.lanes * parts - 1) / (p.lanes * parts);
    // Chunks of up to 128 entries (each leaves up to two partial rows), as many as
    // fill the 24 warps that fit an SM a whole number of times.
    const int64_t groups = static_cast<int64_t>(ctx->sm_count) * 24 * 32 / p.lanes;
    const int64_t work = static_cast<int64_t>(n) * parts;
    const int64_t turns = (work + 128 * groups - 1) / (128 * groups);
    p.chunk = std::max(16, static_cast<int>((work + turns * groups - 1) / std::max<int64_t>(1, turns * groups) + 3) / 4 * 4);
    p.chunks = (n + p.chunk - 1) / p.chunk;
    return p;
}

template <int kSteps>
int launch_scatter(BulletOuCudaCppContext* ctx, const LaunchShape& shape, const SortPass& s) {
    auto with = [&](auto kernel) { return launch_kernel(ctx, "embedding sort launch", kernel, shape, s); };
    if (s.bins <= kThreads) return with(sort_scatter_kernel<kSteps, 1>);
    if (s.bins <= 2 * kThreads) return with(sort_scatter_kernel<kSteps, 2>);
    if (s.bins <= 4 * kThreads) return with(sort_scatter_kernel<kSteps, 4>);
    return with(sort_scatter_kernel<kSteps, 8>);
}

// Sorts the tokens into the scratch at `base`.
int sort_tokens(BulletOuCudaCppContext* ctx, const Tokens& tokens, const GradientPlan& plan, int* base, GradientArgs* out) {
    SortPass s{};
    s.tokens = tokens;
    s.n = tokens.n;
    s.tiles = plan.tiles;
    s.bins = 1 << plan.digit_bits;
    s.totals = base + 4 * plan.row;
    s.counts = s.totals + kMaxBins;
    s.out = reinterpret_cast<int2*>(base);
    if (tokens.n <= kRankMost) {
        const LaunchShape shape{dim3((tokens.n + kRankTokens - 1) / kRankTokens), kThreads, (static_cast<size_t>(tokens.n) + 3) / 4 * 16};
        out->entries = s.out;
        return launch_kernel(ctx, "embedding sort launch", rank_tokens_kernel, shape, tokens, s.out);
    }
    int2* other = s.out + plan.row;
    LaunchShape shape{dim3(plan.tiles), kThreads};
    constexpr int kSteps = kMaxTile / kThreads;
    const int part = kMaxTile / plan.tile;  // the steps of a tile are those of the largest, or a half or a quarter of them
    for (int pass = 0; pass < plan.passes; ++pass) {
        s.shift = pass * plan.digit_bits;
        shape.chained = pass > 0;
        shape.smem = 0;
        shape.grid = dim3(plan.tiles);
        auto* const count = part == 1 ? sort_count_kernel<kSteps> : part == 2 ? sort_count_kernel<kSteps / 2> : sort_count_kernel<kSteps / 4>;
        if (launch_kernel(ctx, "embedding sort launch", count, shape, s) != 0) return -1;
        shape.chained = true;
        shape.grid = dim3(s.bins);
        if (launch_kernel(ctx, "embedding sort launch", sort_scan_kernel, shape, s) != 0) return -1;
        shape.grid = dim3(plan.tiles);
        shape.smem = static_cast<size_t>(kWarps) * s.bins * sizeof(int);
        if ((part == 1   ? launch_scatter<kSteps>(ctx, shape, s)
             : part == 2 ? launch_scatter<kSteps / 2>(ctx, shape, s)
                         : launch_scatter<kSteps / 4>(ctx, shape, s)) != 0)
            return -1;
        s.in = s.out;
        std::swap(s.out, other);
    }
    out->entries = s.in;
    return 0;
}

template <typename In, typename Out, int kUnit, int kLanes, int kUnits>
int launch_gradient(BulletOuCudaCppContext* ctx, const GradientArgs& a) {
    const int per_block = kThreads / kLanes;
    const int64_t blocks = static_cast<int64_t>(a.row_blocks) + (a.chunks + per_block - 1) / per_block;
    if (blocks > INT32_MAX) return fail_message("embedding gradient: too many tokens and rows");
    const int parts = (a.width / kUnit + kLanes * kUnits - 1) / (kLanes * kUnits);
    if (parts > 65535) return fail_messagef("embedding gradient: rows of %d are too wide", a.width);
    LaunchShape shape{dim3(static_cast<unsigned>(blocks), parts), kThreads};
    shape.chained = a.n > 0;
    if (launch_kernel(ctx, "embedding gradient launch", gradient_kernel<In, Out, kUnit, kLanes, kUnits>, shape, a) != 0) return -1;
    if (a.chunks <= 1) return 0;
    LaunchShape join{dim3((a.chunks + kWarps - 1) / kWarps), kThreads};
    join.chained = true;
    return launch_kernel(ctx, "embedding gradient join launch", joined_rows_kernel<Out, kUnit % 4 == 0>, join, a);
}

template <typename In, typename Out, int kUnit>
int launch_gradient_unit(BulletOuCudaCppContext* ctx, const GradientArgs& a, const GradientPlan& p) {
    if (p.lanes == 4) return launch_gradient<In, Out, kUnit, 4, 1>(ctx, a);
    if (p.lanes == 8) return launch_gradient<In, Out, kUnit, 8, 1>(ctx, a);
    if (p.lanes == 16) return launch_gradient<In, Out, kUnit, 16, 1>(ctx, a);
    if constexpr (kUnit == 1) {
        if (p.units == 5) return launch_gradient<In, Out, 1, 32, 5>(ctx, a);
        if (p.units == 4) return launch_gradient<In, Out, 1, 32, 4>(ctx, a);
        if (p.units == 3) return launch_gradient<In, Out, 1, 32, 3>(ctx, a);
    }
    if constexpr (kUnit <= 4) {
        if (p.units == 2) return launch_gradient<In, Out, kUnit, 32, 2>(ctx, a);
    }
    return launch_gradient<In, Out, kUnit, 32, 1>(ctx, a);
}

template <typename In, typename Out>
int gradient(BulletOuCudaCppContext* ctx, const Tokens& t, GradientArgs a, bool vector) {
    const GradientPlan p = plan_gradient(ctx, t.n, t.vocab, a.width, kVectorUnit<In, Out>, vector);
    if (t.n > 0) {
        void* scratch = nullptr;
        if (scratch_slot(ctx, kScratchEmbedding, p.words() * sizeof(int), &scratch, "cudaMalloc embedding gradient") != 0) return -1;
        int* const base = static_cast<int*>(scratch);
        a.heads = reinterpret_cast<float*>(base + 4 * p.row + kMaxBins + p.counts);
        a.tails = a.heads + static_cast<size_t>(p.chunks) * p.width;
        a.part_stride = p.width;
        if (sort_tokens(ctx, t, p, base, &a) != 0) return -1;
    }
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.row_blocks = static_cast<int>((static_cast<int64_t>(a.vocab) + kEmptyRows - 1) / kEmptyRows);
    return vector ? launch_gradient_unit<In, Out, kVectorUnit<In, Out>>(ctx, a, p) : launch_gradient_unit<In, Out, 1>(ctx, a, p);
}

// Whether the rows of both can be taken in units of kUnit elements.
template <typename A, typename B, int kUnit>
bool rows_of_units(const BulletOuB200Matrix& a, const BulletOuB200Matrix& b) {
    return a.cols % kUnit == 0 && rows_aligned(a, std::min<size_t>(16, kUnit * sizeof(A))) &&
           rows_aligned(b, std::min<size_t>(16, kUnit * sizeof(B)));
}

template <typename In, typename Out, int kUnit, int kCols, bool kAnyScale = false>
int launch_lookup(BulletOuCudaCppContext* ctx, const LookupArgs& a) {
    const int units = a.width / kUnit;
    int group = 1;
    while (group < 32 && group < units) group *= 2;
    // as many rows for a group as leave every resident group its share; where
    // the rows are few, their columns are shared too
    const int64_t resident = static_cast<int64_t>(ctx->sm_count) * kLookupCtas;
    int span = 1;
    while (span < group && resident * (kThreads / group) * span < a.tokens.n) span *= 2;
    const int64_t blocks = ((static_cast<int64_t>(a.tokens.n) + span - 1) / span * group + kThreads - 1) / kThreads;
    const unsigned x = static_cast<unsigned>(std::min(blocks, resident));
    const unsigned y = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(units / 64, resident / x)));
    return launch_kernel(ctx, "embedding lookup launch", lookup_kernel<In, Out, kUnit, kCols, kAnyScale>, LaunchShape{dim3(x, y), kThreads}, a, group, span);
}

template <typename In, typename Out>
int lookup(BulletOuCudaCppContext* ctx, const LookupArgs& a, const BulletOuB200Matrix& table, const BulletOuB200Matrix& out) {
    if (!std::isfinite(a.scale)) return launch_lookup<In, Out, 1, 1, true>(ctx, a);
    if (rows_of_units<In, Out, kVectorUnit<In, Out>>(table, out)) return launch_lookup<In, Out, kVectorUnit<In, Out>, 1>(ctx, a);
    if (rows_of_units<In, Out, 2>(table, out))
        return a.width > 64 ? launch_lookup<In, Out, 2, 2>(ctx, a) : launch_lookup<In, Out, 2, 1>(ctx, a);
    if (a.width > 64) return launch_lookup<In, Out, 1, 4>(ctx, a);
    return a.width > 32 ? launch_lookup<In, Out, 1, 2>(ctx, a) : launch_lookup<In, Out, 1, 1>(ctx, a);
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
    const bool in16 = table->type == BULLETOU_B200_TYPE_BF16, out16 = out->type == BULLETOU_B200_TYPE_BF16;
    using B = __nv_bfloat16;
    const int rc = in16 ? (out16 ? lookup<B, B>(ctx, a, *table, *out) : lookup<B, float>(ctx, a, *table, *out))
                        : (out16 ? lookup<float, B>(ctx, a, *table, *out) : lookup<float, float>(ctx, a, *table, *out));
    return rc != 0 ? rc : ok();
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
    const BulletOuB200Matrix &g = *out_gradients, &o = *table_gradients;
    const int rc = in16 ? (out16 ? gradient<B, B>(ctx, t, a, rows_of_units<B, B, kVectorUnit<B, B>>(g, o)) : gradient<B, float>(ctx, t, a, rows_of_units<B, float, kVectorUnit<B, float>>(g, o)))
                        : (out16 ? gradient<float, B>(ctx, t, a, rows_of_units<float, B, kVectorUnit<float, B>>(g, o)) : gradient<float, float>(ctx, t, a, rows_of_units<float, float, kVectorUnit<float, float>>(g, o)));
    return rc != 0 ? rc : ok();
}

}  // extern "C"
