// Router of a mixture of LayerStacks: softmax, top-k, counts of each expert,
// balance loss, and the gradient (sm_100a).
//
// Row t with logits z:   p = softmax(z);  the k largest are chosen;  g = p at
// the chosen, with normalisation g / sum g = softmax over the chosen.
// Over the rows: c_e = choices of e, f_e = c_e / sum c, P_e = sum_t p_te / rows
// alive, loss = balance * E * sum_e f_e P_e.
// Gradient with u = dL/dg and h_e = balance * E * f_e / rows * dL/dloss:
//   plain gates       dz = p * (h + u - sum p (h + u))         (u at the chosen)
//   normalised gates  dz = p * (h - sum p h) + g * (u - sum g u)
// A row is read once in each direction and held in registers.  Sums over a row
// are trees over the lanes that share it; the sums over rows are added up per
// lane, warp and CTA and joined in a fixed order, so no result depends on
// timing.  Counts are integers.
//
// 262144 rows of 81 with their top 2: forward 32 us with the join's launch (the 16
// warps that fit an SM wait for their loads; the comparisons of the maximum and
// the choices, which run at half rate, take 48 % of their pipe), backward 35 us (170
// MB, 4.8 TB/s).  A lane for each row, the rows in shared memory, took 38 and 57 us:
// 20 warps fit an SM, and the shared memory's bandwidth bounds them.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "device_matrix.cuh"
#include "token_launch.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
// By the places of a lane: CTAs on an SM of the backward pass, and threads of the
// forward pass's one CTA on an SM (each CTA leaves sums to be joined): 64
// registers for each thread, 80 for 16 places, up to 128 beyond.
template <int kPlaces>
constexpr int kCtas = kPlaces > 16 ? 2 : kPlaces > 12 ? 3 : 4;
template <int kGroup, int kPlaces>  // (the sums of 512 experts for each warp fill the shared memory)
constexpr int kForwardThreads = kThreads * (kGroup * kPlaces > 256 ? 2 : kCtas<kPlaces>);
constexpr int kMaxExperts = BULLETOU_B200_ROUTER_MAX_EXPERTS;
constexpr int kMaxTopK = BULLETOU_B200_ROUTER_MAX_TOP_K;
constexpr int kJoinThreads = 1024;

struct RouterArgs {
    const void* logits;
    size_t logit_stride;
    int rows, experts, top_k;
    float balance;
    int normalize;
    int* chosen;
    size_t chosen_stride;
    float* gates;
    size_t gate_stride;
    int* counts;
    float* mean;
    float* loss;
    // per CTA: probability sums [grid][experts], counts [grid][experts + 1]
    float* part_p;
    int* part_c;
    // backward
    const float* gate_grad;
    size_t gate_grad_stride;
    const float* loss_grad;
    void* logit_grad;
    size_t logit_grad_stride;
};

// 2^x to about two units in the last place, and a maximum that keeps NaN.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float2 b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b.x), "f"(b.y));
    return y;
}
// 1 / x of a row's sums: the approximation and a step of Newton's iteration, half a
// unit in the last place.  CUDA's division, whose special cases do not occur here,
// takes 3 us more forward and 2 backward for 262144 x 81.
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return __fmaf_rn(y, __fmaf_rn(-x, y, 1.0f), y);
}
// A gate's part of its row's, corrected by its remainder; exactly one where it is
// the only one.
__device__ __forceinline__ float share_of(float p, float total) {
    const float inverse = reciprocal(total), q = p * inverse;
    return p == total ? 1.0f : __fmaf_rn(__fmaf_rn(-q, total, p), inverse, q);
}
constexpr float kLog2E = 1.4426950408889634f;

// Over the kGroup lanes that share a row.
template <int kGroup>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = kGroup / 2; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
template <int kGroup>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = kGroup / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
template <int kGroup>
__device__ __forceinline__ int group_min(int v) {
#pragma unroll
    for (int d = kGroup / 2; d > 0; d >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

// Two f32 operations in one instruction, each rounded as by itself.  (By CUDA's
// __fadd2_rn and its like 262144 x 81 f32 takes 40 us backward, so 37.)
__device__ __forceinline__ uint64_t packed(float2 v) {
    uint64_t u;
    memcpy(&u, &v, sizeof(u));
    return u;
}
__device__ __forceinline__ float2 unpacked(uint64_t u) {
    float2 v;
    memcpy(&v, &u, sizeof(v));
    return v;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(packed(a)), "l"(packed(b)));
    return unpacked(y);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(packed(a)), "l"(packed(b)));
    return unpacked(y);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(packed(a)), "l"(packed(b)), "l"(packed(c)));
    return unpacked(y);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A row's logits and their exponentials: expert e in lane e % kGroup, place
// e / kGroup; only the last two places may lie past the last expert, and hold
// -inf and 0 there.  All lanes of a warp come here together; a row past the end
// is one that is not alive.
//
// exp(z - top) is taken as 2^((z - top) log2 e): two roundings of 2^-24 relative
// in an exponent below 20 wherever p > 10^-6.
template <int kGroup, int kPlaces>
struct Row {
    static_assert(kPlaces % 2 == 0);
    float2 z[kPlaces / 2];
    float2 e[kPlaces / 2];
    float top, shift, inverse;  // p = e * inverse, e = exp(z - shift); shift is top where that is finite
    bool alive;                 // the largest logit is finite

    __device__ __forceinline__ float& logit(int i) { return i % 2 == 0 ? z[i / 2].x : z[i / 2].y; }
    __device__ __forceinline__ float largest() const {
        float m = max_nan(z[0].x, z[0].y);
#pragma unroll
        for (int i = 1; i < kPlaces / 2; ++i) m = max_nan(m, z[i]);
        return m;
    }
    __device__ __forceinline__ float exponential(float logit) const { return exp2_approx((logit - shift) * kLog2E); }

    // `src`: the row's logit in place 0 of this lane; `mine`: the places that it has, 0 in a row past the end.
    template <typename T>
    __device__ __forceinline__ void load(const T* src, int mine) {
        const bool valid = mine > 0;
#pragma unroll
        for (int i = 0; i < kPlaces; ++i)
            logit(i) = (i < kPlaces - 2 ? valid : i < mine) ? to_f32(src[kGroup * i]) : -INFINITY;
    }

    __device__ __forceinline__ void normalise() {
        top = group_max<kGroup>(largest());
        alive = top > -INFINITY && top < INFINITY;
        shift = alive ? top : 0.0f;
        float2 sum = both(0.0f);
#pragma unroll
        for (int i = 0; i < kPlaces / 2; ++i) {
            const float2 x = mul2(add2(z[i], both(-shift)), both(kLog2E));
            e[i] = make_float2(exp2_approx(x.x), exp2_approx(x.y));
            sum = add2(sum, e[i]);
        }
        const float total = group_sum<kGroup>(sum.x + sum.y);
        // a masked row's exponentials are zeros; a broken row is NaN
        inverse = alive ? reciprocal(total) : top == -INFINITY ? 0.0f : NAN;
    }
};

// The places that this lane has in a row of `experts`.
template <int kGroup>
__device__ __forceinline__ int places_of(int experts, int lane) {
    return (experts - lane + kGroup - 1) / kGroup;
}

// The choices of all experts, by the CTA's first warp.
__device__ __forceinline__ void sum_choices(const int* counts, int experts, int64_t* choices) {
    if (threadIdx.x >= 32) return;
    int64_t c = 0;
    for (int e = threadIdx.x; e < experts; e += 32) c += counts[e];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
    if (threadIdx.x == 0) *choices = c;
}

// Means and loss from the sums of the probabilities and the counts; every
// thread of the CTA comes here.
__device__ void finish(const RouterArgs& a, const float* p_sums, const int* counts) {
    __shared__ int64_t choices;
    __shared__ float warp_terms[32];
    sum_choices(counts, a.experts, &choices);
    __syncthreads();
    const float rows = static_cast<float>(max(counts[a.experts], 1)), all = static_cast<float>(max(choices, static_cast<int64_t>(1)));
    float s = 0.0f;
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
        const float mean = p_sums[e] / rows;
        a.mean[e] = mean;
        a.counts[e] = counts[e];
        s += static_cast<float>(counts[e]) / all * mean;
    }
    if (threadIdx.x == 0) a.counts[a.experts] = counts[a.experts];
    s = group_sum<32>(s);
    if ((threadIdx.x & 31) == 0) warp_terms[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        float total = 0.0f;
        for (unsigned w = 0; w < blockDim.x / 32; ++w) total += warp_terms[w];
        a.loss[0] = a.balance * static_cast<float>(a.experts) * total;
    }
}

// kGroup lanes for each row (at least top_k), kPlaces experts in each lane.  One
// CTA alone also finishes; otherwise the CTAs leave their sums to router_join_kernel.
template <typename T, int kGroup, int kPlaces>
__global__ void __launch_bounds__(kForwardThreads<kGroup, kPlaces>, 1) router_forward_kernel(const RouterArgs a) {
    constexpr int kThreads = kForwardThreads<kGroup, kPlaces>, kWarps = kThreads / 32;
    __shared__ int count[kMaxExperts + 1];
    __shared__ float psum[kWarps][kGroup * kPlaces];
    const int lane = threadIdx.x & (kGroup - 1), warp = threadIdx.x >> 5;
    let_next_start();
    for (int i = threadIdx.x; i <= a.experts; i += kThreads) count[i] = 0;
    __syncthreads();
    float2 acc[kPlaces / 2] = {};
    int alive = 0;
    constexpr int kRows = kThreads / kGroup;
    const int places = places_of<kGroup>(a.experts, lane);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t t = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kGroup;
    const T* src = static_cast<const T*>(a.logits) + t * a.logit_stride + lane;
    int* chosen = a.chosen + t * a.chosen_stride + lane;
    float* gates = a.gates + t * a.gate_stride + lane;
    // (the lanes of a warp stay together for the trees)
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * kRows; t0 < a.rows; t0 += step, t += step) {
        Row<kGroup, kPlaces> r;
        r.template load<T>(src, t < a.rows ? places : 0);
        r.normalise();
#pragma unroll
        for (int i = 0; i < kPlaces / 2; ++i) acc[i] = fma2(r.e[i], both(r.inverse), acc[i]);
        alive += r.alive && lane == 0;
        float total = 0.0f, own = 0.0f;  // lane j keeps the j-th choice
        int pick = -1;
        float best = r.top;
        for (int j = 0;;) {
            int at = kMaxExperts;  // the lowest index that has the largest logit left
#pragma unroll
            for (int i = kPlaces - 1; i >= 0; --i)
                if (r.logit(i) == best) at = lane + kGroup * i;
            at = group_min<kGroup>(at);
            const bool some = r.alive && best > -INFINITY;
            const float gate = some ? r.exponential(best) * r.inverse : 0.0f;
            total += gate;
            if (j == lane) {
                pick = some ? at : -1;
                own = gate;
            }
            if (++j >= a.top_k) break;
#pragma unroll
            for (int i = 0; i < kPlaces; ++i)
                if (lane + kGroup * i == at) r.logit(i) = -INFINITY;
            best = group_max<kGroup>(r.largest());
        }
        if (lane < a.top_k && t < a.rows) {
            *chosen = pick;
            *gates = a.normalize && pick >= 0 ? share_of(own, total) : own;
            if (pick >= 0) atomicAdd(count + pick, 1);
        }
        src += step * a.logit_stride;
        chosen += step * a.chosen_stride;
        gates += step * a.gate_stride;
    }
    if (alive != 0) atomicAdd(count + a.experts, alive);
#pragma unroll
    for (int i = 0; i < kPlaces; ++i) {
        float s = i % 2 == 0 ? acc[i / 2].x : acc[i / 2].y;
#pragma unroll
        for (int d = kGroup; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if ((threadIdx.x & 31) < kGroup) psum[warp][lane + kGroup * i] = s;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        float s = 0.0f;
        for (int w = 0; w < kWarps; ++w) s += psum[w][e];
        if (gridDim.x == 1) psum[0][e] = s;
        else a.part_p[static_cast<size_t>(blockIdx.x) * a.experts + e] = s;
    }
    __syncthreads();
    if (gridDim.x == 1) {
        finish(a, psum[0], count);
        return;
    }
    for (int e = threadIdx.x; e <= a.experts; e += kThreads)
        a.part_c[static_cast<size_t>(blockIdx.x) * (a.experts + 1) + e] = count[e];
}

// One CTA: the CTAs' sums joined, each warp every 32nd of them, then the warps
// in order.
__global__ void __launch_bounds__(kJoinThreads) router_join_kernel(const RouterArgs a, int parts) {
    constexpr int kJoinWarps = kJoinThreads / 32, kAtOnce = 128;
    __shared__ float part[kJoinWarps][kAtOnce];
    __shared__ float p_sums[kMaxExperts];
    __shared__ int count[kMaxExperts + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= a.experts; e += kJoinThreads) count[e] = 0;
    __syncthreads();
    wait_for_previous();
    for (int e0 = 0; e0 <= a.experts; e0 += kAtOnce) {
        float p[kAtOnce / 32] = {};
        int c[kAtOnce / 32] = {};
        for (int i0 = warp; i0 < parts; i0 += 4 * kJoinWarps) {
            float pv[4][kAtOnce / 32];
            int cv[4][kAtOnce / 32];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int i = i0 + b * kJoinWarps;
#pragma unroll
                for (int j = 0; j < kAtOnce / 32; ++j) {
                    const int e = e0 + lane + 32 * j;
                    pv[b][j] = i < parts && e < a.experts ? a.part_p[static_cast<size_t>(i) * a.experts + e] : 0.0f;
                    cv[b][j] = i < parts && e <= a.experts ? a.part_c[static_cast<size_t>(i) * (a.experts + 1) + e] : 0;
                }
            }
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int j = 0; j < kAtOnce / 32; ++j) {
                    p[j] += pv[b][j];
                    c[j] += cv[b][j];
                }
        }
#pragma unroll
        for (int j = 0; j < kAtOnce / 32; ++j) {
            part[warp][lane + 32 * j] = p[j];
            if (c[j] != 0) atomicAdd(count + e0 + lane + 32 * j, c[j]);
        }
        __syncthreads();
        if (threadIdx.x < kAtOnce && e0 + static_cast<int>(threadIdx.x) < a.experts) {
            float s = 0.0f;
            for (int w = 0; w < kJoinWarps; ++w) s += part[w][threadIdx.x];
            p_sums[e0 + threadIdx.x] = s;
        }
        __syncthreads();
    }
    finish(a, p_sums, count);
}

template <typename T, int kGroup, int kPlaces>
__global__ void __launch_bounds__(kThreads, kCtas<kPlaces>) router_backward_kernel(const RouterArgs a) {
    __shared__ int64_t choices;
    __shared__ int shared_counts[kGroup * kPlaces];
    __shared__ float shared_pull[kGroup * kPlaces];
    const int lane = threadIdx.x & (kGroup - 1);
    for (int e = threadIdx.x; e < kGroup * kPlaces; e += kThreads) shared_counts[e] = e < a.experts ? a.counts[e] : 0;
    __syncthreads();
    sum_choices(shared_counts, a.experts, &choices);
    __syncthreads();
    // The balance loss's pull on every probability of an expert, h_e less the mean
    // of h: the probabilities sum to one, so what all h share cancels, and experts
    // nearly in balance would leave only its rounding.  E c_e - sum c is exact.
    const float unit = (a.loss_grad != nullptr ? a.loss_grad[0] : 0.0f) * a.balance / static_cast<float>(max(a.counts[a.experts], 1)) /
                       static_cast<float>(max(choices, static_cast<int64_t>(1)));
    for (int e = threadIdx.x; e < kGroup * kPlaces; e += kThreads)
        shared_pull[e] = e < a.experts ? static_cast<float>(static_cast<int64_t>(shared_counts[e]) * a.experts - choices) * unit : 0.0f;
    __syncthreads();
    float2 h[kPlaces / 2];
#pragma unroll
    for (int i = 0; i < kPlaces / 2; ++i) h[i] = make_float2(shared_pull[lane + kGroup * 2 * i], shared_pull[lane + kGroup * (2 * i + 1)]);
    constexpr int kRows = kThreads / kGroup;
    const int places = places_of<kGroup>(a.experts, lane);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
    int64_t t = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kGroup;
    const T* src = static_cast<const T*>(a.logits) + t * a.logit_stride + lane;
    T* dst = static_cast<T*>(a.logit_grad) + t * a.logit_grad_stride + lane;
    const int* chosen = a.chosen + t * a.chosen_stride + lane;
    const float* gate_grad = a.gate_grad + t * a.gate_grad_stride + lane;
    // lane j holds the j-th choice and its gate's gradient, of the next row already
    const bool chooses = a.gate_grad != nullptr && lane < a.top_k;
    int next_pick = chooses && t < a.rows ? *chosen : -1;
    float next_up = chooses && t < a.rows ? *gate_grad : 0.0f;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * kRows; t0 < a.rows; t0 += step, t += step) {
        const int mine = t < a.rows ? places : 0;
        const int pick = next_pick >= 0 && next_pick < a.experts ? next_pick : -1;
        const float up = pick >= 0 ? next_up : 0.0f;
        Row<kGroup, kPlaces> r;
        r.template load<T>(src, mine);
        const float z = pick >= 0 ? to_f32(src[pick - lane]) : -INFINITY;
        const float pull = pick >= 0 ? shared_pull[pick] : 0.0f;
        chosen += step * a.chosen_stride;
        gate_grad += step * a.gate_grad_stride;
        next_pick = chooses && t + step < a.rows ? *chosen : -1;
        next_up = chooses && t + step < a.rows ? *gate_grad : 0.0f;
        r.normalise();
        const float p = pick >= 0 ? r.exponential(z) * r.inverse : 0.0f;
        float2 dots = both(0.0f);
#pragma unroll
        for (int i = 0; i < kPlaces / 2; ++i) {
            r.e[i] = mul2(r.e[i], both(r.inverse));
            dots = fma2(r.e[i], h[i], dots);
        }
        float dot = group_sum<kGroup>(dots.x + dots.y);
        float direct = 0.0f;  // what the choice's gate adds to its logit's gradient
        if (a.gate_grad != nullptr) {
            if (a.normalize) {
                // g (u - sum g u): gates that sum to one take no part in the mean, and a
                // single one adds nothing
                const float total = group_sum<kGroup>(p);
                const float gate = total > 0.0f ? share_of(p, total) : 0.0f;
                direct = gate * (up - group_sum<kGroup>(gate * up));
            } else {
                direct = p * up;
                dot += group_sum<kGroup>(direct);
            }
        }
#pragma unroll
        for (int i = 0; i < kPlaces / 2; ++i) {
            const float2 g = mul2(r.e[i], add2(h[i], both(-dot)));
            if (2 * i < kPlaces - 2 ? mine > 0 : 2 * i < mine) dst[kGroup * 2 * i] = from_f32<T>(g.x);
            if (2 * i < kPlaces - 2 ? mine > 0 : 2 * i + 1 < mine) dst[kGroup * (2 * i + 1)] = from_f32<T>(g.y);
        }
        __syncwarp();  // the chosen ones are written again, after the lane that had them
        if (pick >= 0) dst[pick - lane] = from_f32<T>(__fmaf_rn(p, pull - dot, direct));
        src += step * a.logit_stride;
        dst += step * a.logit_grad_stride;
    }
}

int validate_counts(const RouterArgs& a) {
    if (a.experts < 1 || a.experts > kMaxExperts)
        return fail_messagef("router: %d experts, 1 to %d are supported", a.experts, kMaxExperts);
    if (a.top_k < 1 || a.top_k > kMaxTopK || a.top_k > a.experts)
        return fail_messagef("router: top_k %d, 1 to %d and at most the %d experts are supported", a.top_k, kMaxTopK,
                             a.experts);
    return 0;
}

// The lanes of a row, at least one for every choice, and the places of a lane, at
// most two more than the experts need.  Forward, few lanes: the trees over lanes
// are short and the rest is a lane's own work (262144 x 81, top 2: 4 lanes 27 us,
// 8 lanes 32 us).  Backward, every place is a store, whose sectors the lanes of a
// row should fill (4 lanes 45 us, 8 lanes 36 us, 16 lanes 44 us; at 128 experts 8
// lanes 13.5 us, 16 lanes 12.3 us for 65536 rows).
template <int kGroup, int kPlaces, typename F>
int with_places(const RouterArgs& a, F&& f) {
    if constexpr (kPlaces > 2)
        if (a.experts <= kGroup * (kPlaces - 2)) return with_places<kGroup, kPlaces - 2>(a, f);
    return f(std::integral_constant<int, kGroup>{}, std::integral_constant<int, kPlaces>{});
}
template <typename F>
int with_forward_shape(const RouterArgs& a, F&& f) {
    if (a.experts <= 96 && a.top_k <= 4) return with_places<4, 24>(a, f);
    if (a.experts <= 128) return with_places<8, 16>(a, f);
    if (a.experts <= 256) return with_places<16, 16>(a, f);
    return with_places<32, 16>(a, f);
}
template <typename F>
int with_backward_shape(const RouterArgs& a, F&& f) {
    if (a.experts <= 16 && a.top_k <= 4) return with_places<4, 4>(a, f);
    if (a.experts <= 96) return with_places<8, 12>(a, f);
    if (a.experts <= 128) return with_places<16, 8>(a, f);
    return with_places<32, 16>(a, f);
}

// CTAs for the rows; up to two rounds of rows are left to one CTA, which then
// needs no second launch.
int router_grid(const BulletOuCudaCppContext* ctx, int rows, int per) {
    const int64_t ctas = (static_cast<int64_t>(rows) + per - 1) / per;
    return ctas <= 2 ? 1 : static_cast<int>(std::min<int64_t>(ctas, ctx->sm_count));
}

template <typename T>
int forward(BulletOuCudaCppContext* ctx, RouterArgs a) {
    return with_forward_shape(a, [&](auto group, auto places) {
        const int grid = router_grid(ctx, a.rows, kForwardThreads<group(), places()> / group());
        if (grid > 1) {
            void* p = nullptr;
            if (scratch_slot(ctx, kScratchRouter, static_cast<size_t>(grid) * (2 * a.experts + 1) * 4, &p,
                             "cudaMalloc router parts") != 0)
                return -1;
            a.part_p = static_cast<float*>(p);
            a.part_c = static_cast<int*>(p) + static_cast<size_t>(grid) * a.experts;
        }
        LaunchShape shape{dim3(grid), kForwardThreads<group(), places()>};
        if (launch_kernel(ctx, "router forward launch", router_forward_kernel<T, group(), places()>, shape, a) != 0) return -1;
        if (grid == 1) return 0;
        LaunchShape join{dim3(1), kJoinThreads};
        join.chained = true;
        return launch_kernel(ctx, "router join launch", router_join_kernel, join, a, grid);
    });
}

template <typename T>
int backward(BulletOuCudaCppContext* ctx, const RouterArgs& a) {
    return with_backward_shape(a, [&](auto group, auto places) {
        const int64_t ctas = (static_cast<int64_t>(a.rows) * group + kThreads - 1) / kThreads;
        const LaunchShape shape{dim3(static_cast<unsigned>(std::min<int64_t>(ctas, static_cast<int64_t>(ctx->sm_count) * kCtas<places()>))), kThreads};
        return launch_kernel(ctx, "router backward launch", router_backward_kernel<T, group(), places()>, shape, a);
    });
}

}  // namespace
}  // namespace bou

using namespace bou;

extern "C" {

int bulletou_b200_router_forward_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* logits, float balance,
                                        int normalize_gates, const BulletOuB200Matrix* experts,
                                        const BulletOuB200Matrix* gates, const BulletOuB200Matrix* counts,
                                        const BulletOuB200Matrix* mean_probabilities, const BulletOuB200Matrix* loss) {
    if (set_device(ctx) != 0 || validate_matrix(logits, kTypeFloat, "router logits") != 0 ||
        validate_matrix(experts, kTypeI32, "router experts") != 0)
        return -1;
    RouterArgs a{};
    a.rows = static_cast<int>(logits->rows);
    a.experts = static_cast<int>(logits->cols);
    a.top_k = static_cast<int>(experts->cols);
    if (validate_counts(a) != 0 || validate_matrix(experts, kTypeI32, logits->rows, experts->cols, "router experts") != 0 ||
        validate_matrix(gates, kTypeF32, logits->rows, experts->cols, "router gates") != 0 ||
        validate_matrix(counts, kTypeI32, 1, logits->cols + 1, "router counts") != 0 ||
        validate_matrix(mean_probabilities, kTypeF32, 1, logits->cols, "router mean probabilities") != 0 ||
        validate_matrix(loss, kTypeF32, 1, 1, "router loss") != 0)
        return -1;
    const BulletOuB200Matrix* outs[] = {experts, gates, counts, mean_probabilities, loss};
    const char* names[] = {"router experts", "router gates", "router counts", "router mean probabilities", "router loss"};
    for (int i = 0; i < 5; ++i) {
        if (validate_disjoint(outs[i], names[i], logits, "the logits") != 0) return -1;
        for (int j = 0; j < i; ++j)
            if (validate_disjoint(outs[i], names[i], outs[j], names[j]) != 0) return -1;
    }
    a.logits = logits->data;
    a.logit_stride = logits->row_stride;
    a.balance = balance;
    a.normalize = normalize_gates != 0;
    a.chosen = static_cast<int*>(experts->data);
    a.chosen_stride = experts->row_stride;
    a.gates = static_cast<float*>(gates->data);
    a.gate_stride = gates->row_stride;
    a.counts = static_cast<int*>(counts->data);
    a.mean = static_cast<float*>(mean_probabilities->data);
    a.loss = static_cast<float*>(loss->data);
    const int rc = logits->type == BULLETOU_B200_TYPE_F32 ? forward<float>(ctx, a) : forward<__nv_bfloat16>(ctx, a);
    return rc != 0 ? rc : ok();
}

int bulletou_b200_router_backward_device(BulletOuCudaCppContext* ctx, const BulletOuB200Matrix* logits,
                                         const BulletOuB200Matrix* experts, const BulletOuB200Matrix* counts,
                                         const BulletOuB200Matrix* gate_gradients,
                                         const BulletOuB200Matrix* loss_gradient, float balance, int normalize_gates,
                                         const BulletOuB200Matrix* logit_gradients) {
    if (set_device(ctx) != 0 || validate_matrix(logits, kTypeFloat, "router logits") != 0 ||
        validate_matrix(experts, kTypeI32, "router experts") != 0)
        return -1;
    RouterArgs a{};
    a.rows = static_cast<int>(logits->rows);
    a.experts = static_cast<int>(logits->cols);
    a.top_k = static_cast<int>(experts->cols);
    if (validate_counts(a) != 0 || validate_matrix(experts, kTypeI32, logits->rows, experts->cols, "router experts") != 0 ||
        validate_matrix(counts, kTypeI32, 1, logits->cols + 1, "router counts") != 0 ||
        (gate_gradients != nullptr &&
         validate_matrix(gate_gradients, kTypeF32, logits->rows, experts->cols, "router gate gradients") != 0) ||
        (loss_gradient != nullptr && validate_matrix(loss_gradient, kTypeF32, 1, 1, "router loss gradient") != 0) ||
        validate_matrix(logit_gradients, 1u << logits->type, logits->rows, logits->cols, "router logit gradients") != 0 ||
        validate_disjoint(logit_gradients, "router logit gradients", logits, "the logits", true) != 0 ||
        validate_disjoint(logit_gradients, "router logit gradients", experts, "the experts") != 0 ||
        validate_disjoint(logit_gradients, "router logit gradients", counts, "the counts") != 0 ||
        validate_disjoint(logit_gradients, "router logit gradients", gate_gradients, "the gate gradients") != 0 ||
        validate_disjoint(logit_gradients, "router logit gradients", loss_gradient, "the loss gradient") != 0)
        return -1;
    if (a.rows == 0) return ok();
    a.logits = logits->data;
    a.logit_stride = logits->row_stride;
    a.balance = balance;
    a.normalize = normalize_gates != 0;
    a.chosen = static_cast<int*>(experts->data);
    a.chosen_stride = experts->row_stride;
    a.counts = static_cast<int*>(counts->data);
    a.gate_grad = gate_gradients != nullptr ? static_cast<const float*>(gate_gradients->data) : nullptr;
    a.gate_grad_stride = gate_gradients != nullptr ? gate_gradients->row_stride : 0;
    a.loss_grad = loss_gradient != nullptr ? static_cast<const float*>(loss_gradient->data) : nullptr;
    a.logit_grad = logit_gradients->data;
    a.logit_grad_stride = logit_gradients->row_stride;
    const int rc = logits->type == BULLETOU_B200_TYPE_F32 ? backward<float>(ctx, a) : backward<__nv_bfloat16>(ctx, a);
    return rc != 0 ? rc : ok();
}

}  // extern "C"
