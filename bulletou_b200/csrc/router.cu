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
// Sums over a row are trees over a warp's lanes; the sums over rows are added
// up per lane, warp and CTA and joined in a fixed order, so no result depends
// on timing.  Counts are integers.
#include <algorithm>

#include "device_matrix.cuh"

namespace bou {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = BULLETOU_B200_ROUTER_MAX_EXPERTS;
constexpr int kMaxTopK = BULLETOU_B200_ROUTER_MAX_TOP_K;
constexpr int kPerLane = kMaxExperts / 32;

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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// A row's logits and probabilities, expert e in lane e % 32, place e / 32.
struct Row {
    float z[kPerLane];
    float p[kPerLane];
    bool alive;  // the largest logit is finite
};

template <typename T>
__device__ __forceinline__ void load_row(const RouterArgs& a, int t, int lane, Row& r) {
    const T* src = static_cast<const T*>(a.logits) + t * a.logit_stride;
    float top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int e = lane + 32 * i;
        r.z[i] = e < a.experts ? to_f32(src[e]) : -INFINITY;
        nan |= r.z[i] != r.z[i];
        top = fmaxf(top, r.z[i]);
    }
    nan = __any_sync(0xffffffffu, nan);
    top = warp_max(top);
    r.alive = !nan && top > -INFINITY && top < INFINITY;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        r.p[i] = r.alive ? expf(r.z[i] - top) : 0.0f;
        sum += r.p[i];
    }
    sum = warp_sum(sum);
    const float broken = (nan || top == INFINITY) ? NAN : 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const bool used = lane + 32 * i < a.experts;
        r.p[i] = r.alive ? r.p[i] / sum : (used ? broken : 0.0f);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) router_forward_kernel(const RouterArgs a) {
    __shared__ int count[kMaxExperts + 1];
    __shared__ float psum[kWarps][kMaxExperts];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i <= a.experts; i += kThreads) count[i] = 0;
    __syncthreads();
    float acc[kPerLane] = {};
    for (int t = blockIdx.x * kWarps + warp; t < a.rows; t += gridDim.x * kWarps) {
        Row r;
        load_row<T>(a, t, lane, r);
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) acc[i] += r.p[i];
        int pick[kMaxTopK];
        float gate[kMaxTopK];
        float total = 0.0f;
#pragma unroll
        for (int j = 0; j < kMaxTopK; ++j) {
            if (j >= a.top_k) break;
            float best = -INFINITY, best_p = 0.0f;
            int at = kMaxExperts;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (r.z[i] > best) {
                    best = r.z[i];
                    best_p = r.p[i];
                    at = lane + 32 * i;
                }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                const float z = __shfl_xor_sync(0xffffffffu, best, d);
                const float p = __shfl_xor_sync(0xffffffffu, best_p, d);
                const int e = __shfl_xor_sync(0xffffffffu, at, d);
                if (z > best || (z == best && e < at)) {
                    best = z;
                    best_p = p;
                    at = e;
                }
            }
            const bool some = r.alive && best > -INFINITY;
            pick[j] = some ? at : -1;
            gate[j] = some ? best_p : 0.0f;
            total += gate[j];
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (lane + 32 * i == at) r.z[i] = -INFINITY;
        }
        if (lane == 0) {
            if (r.alive) atomicAdd(count + a.experts, 1);
            for (int j = 0; j < kMaxTopK; ++j) {
                if (j >= a.top_k) break;
                if (pick[j] >= 0) atomicAdd(count + pick[j], 1);
                a.chosen[t * a.chosen_stride + j] = pick[j];
                a.gates[t * a.gate_stride + j] = a.normalize && pick[j] >= 0 ? gate[j] / total : gate[j];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) psum[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        float s = 0.0f;
        for (int w = 0; w < kWarps; ++w) s += psum[w][e];
        a.part_p[static_cast<size_t>(blockIdx.x) * a.experts + e] = s;
    }
    for (int e = threadIdx.x; e <= a.experts; e += kThreads)
        a.part_c[static_cast<size_t>(blockIdx.x) * (a.experts + 1) + e] = count[e];
}

// One CTA: the CTAs' parts joined in order, means and loss.
__global__ void __launch_bounds__(kMaxExperts) router_join_kernel(const RouterArgs a, int parts) {
    __shared__ float term[kMaxExperts];
    __shared__ int rows, choices;
    if (threadIdx.x == 0) rows = choices = 0;
    __syncthreads();
    float p = 0.0f;
    int c = 0;
    const int e = threadIdx.x;
    if (e < a.experts)
        for (int i = 0; i < parts; ++i) {
            p += a.part_p[static_cast<size_t>(i) * a.experts + e];
            c += a.part_c[static_cast<size_t>(i) * (a.experts + 1) + e];
        }
    atomicAdd(&choices, c);
    int r = 0;
    for (int i = threadIdx.x; i < parts; i += kMaxExperts) r += a.part_c[static_cast<size_t>(i) * (a.experts + 1) + a.experts];
    atomicAdd(&rows, r);
    __syncthreads();
    const float mean = p / static_cast<float>(max(rows, 1));
    term[e] = 0.0f;
    if (e < a.experts) {
        a.mean[e] = mean;
        a.counts[e] = c;
        term[e] = static_cast<float>(c) / static_cast<float>(max(choices, 1)) * mean;
    }
    if (e == 0) a.counts[a.experts] = rows;
    __syncthreads();
    for (int d = kMaxExperts / 2; d > 0; d >>= 1) {
        if (e < d) term[e] += term[e + d];
        __syncthreads();
    }
    if (e == 0) a.loss[0] = a.balance * static_cast<float>(a.experts) * term[0];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) router_backward_kernel(const RouterArgs a) {
    __shared__ int choices;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) choices = 0;
    __syncthreads();
    int c = 0;
    for (int e = threadIdx.x; e < a.experts; e += kThreads) c += a.counts[e];
    atomicAdd(&choices, c);
    __syncthreads();
    // the balance loss's pull on every probability of an expert
    float h[kPerLane];
    const float unit = (a.loss_grad != nullptr ? a.loss_grad[0] : 0.0f) * a.balance * static_cast<float>(a.experts) /
                       static_cast<float>(max(a.counts[a.experts], 1));
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int e = lane + 32 * i;
        h[i] = e < a.experts ? static_cast<float>(a.counts[e]) / static_cast<float>(max(choices, 1)) * unit : 0.0f;
    }
    for (int t = blockIdx.x * kWarps + warp; t < a.rows; t += gridDim.x * kWarps) {
        Row r;
        load_row<T>(a, t, lane, r);
        float u[kPerLane], g[kPerLane];  // gate gradients and gates at the chosen experts
        float total = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) u[i] = g[i] = 0.0f;
        if (a.gate_grad != nullptr)
            for (int j = 0; j < a.top_k; ++j) {
                const int e = a.chosen[t * a.chosen_stride + j];
                if (e < 0 || e >= a.experts) continue;
                const float up = a.gate_grad[t * a.gate_grad_stride + j];
#pragma unroll
                for (int i = 0; i < kPerLane; ++i)
                    if (lane + 32 * i == e) {
                        u[i] = up;
                        g[i] = r.p[i];
                    }
            }
        if (a.normalize && a.gate_grad != nullptr) {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) total += g[i];
            total = warp_sum(total);
            float own = 0.0f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                g[i] = total > 0.0f ? g[i] / total : 0.0f;
                own += g[i] * u[i];
            }
            own = warp_sum(own);
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                g[i] *= u[i] - own;  // the part through the gates
                u[i] = 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) g[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) dot += r.p[i] * (h[i] + u[i]);
        dot = warp_sum(dot);
        T* dst = static_cast<T*>(a.logit_grad) + t * a.logit_grad_stride;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int e = lane + 32 * i;
            if (e < a.experts) dst[e] = from_f32<T>(r.p[i] * (h[i] + u[i] - dot) + g[i]);
        }
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

int router_grid(const BulletOuCudaCppContext* ctx, int rows) {
    return std::max(1, std::min((rows + kWarps - 1) / kWarps, ctx->sm_count * 4));
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
    const int grid = router_grid(ctx, a.rows);
    void* p = nullptr;
    if (scratch_slot(ctx, kScratchRouter, static_cast<size_t>(grid) * (2 * a.experts + 1) * 4, &p,
                     "cudaMalloc router parts") != 0)
        return -1;
    a.part_p = static_cast<float*>(p);
    a.part_c = static_cast<int*>(p) + static_cast<size_t>(grid) * a.experts;
    if (logits->type == BULLETOU_B200_TYPE_F32)
        router_forward_kernel<float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else
        router_forward_kernel<__nv_bfloat16><<<grid, kThreads, 0, ctx->stream>>>(a);
    router_join_kernel<<<1, kMaxExperts, 0, ctx->stream>>>(a, grid);
    return check_launch("router forward launch") != 0 ? -1 : ok();
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
    const int grid = router_grid(ctx, a.rows);
    if (logits->type == BULLETOU_B200_TYPE_F32)
        router_backward_kernel<float><<<grid, kThreads, 0, ctx->stream>>>(a);
    else
        router_backward_kernel<__nv_bfloat16><<<grid, kThreads, 0, ctx->stream>>>(a);
    return check_launch("router backward launch") != 0 ? -1 : ok();
}

}  // extern "C"
