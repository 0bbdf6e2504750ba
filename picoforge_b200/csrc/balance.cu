// The balance loss of a router with per-expert counts, and the gradient of the router's logits (contract:
// include/qwen4_moe_b200.h; no counterpart in the reference).
//
// p = softmax(z) per token; c_e the (token, slot) pairs of expert e, P_e = sum_t p_te, over the N tokens that count;
//   L = E / N^2 sum_e c_e P_e              dL/dz_t = E / N^2 p_t (c - <c, p_t>)
// and of the route weights w of the chosen experts i_1..i_K, for an incoming gradient dw:
//   normalised (w = softmax over the chosen logits)   dz[i_k] += w_k (dw_k - sum_j w_j dw_j)
//   not normalised (w_k = p[i_k])                     dz_e    += p_e ([e = i_k] dw_k - sum_j p[i_j] dw_j)
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "cuda_shim.h"

extern "C" int qw4sh_note_launch(const char *name);
extern "C" int qw4sh_fail_text(const char *text);

namespace {

constexpr float UNIT = 1099511627776.0f;          // 2^40: probability sums meet as 64-bit integers, whose sum has no order

__device__ __forceinline__ float warp_max(float v) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A row that has no softmax is noted with its number (the lowest is kept).
__device__ __noinline__ void note_nonfinite(uint32_t *status, uint32_t row) {
    atomicOr(status, QW4SH_ERR_NONFINITE);
    atomicMin(status + 1, row);
}

// One warp per row, three passes over it (the second and third out of L1).
__global__ void __launch_bounds__(256) balance_forward_kernel(uint32_t E, uint32_t K, const float *__restrict__ logits, uint64_t pitch,
                                                              const uint32_t *__restrict__ ids, const uint8_t *__restrict__ mask, uint32_t T,
                                                              QW4ShTune tune, uint32_t *__restrict__ counts, float *__restrict__ prob_sums,
                                                              float *__restrict__ loss) {
    extern __shared__ uint32_t hist[];            // [E] counts, [E] sums as 64-bit integers
    unsigned long long *sums = (unsigned long long *)(hist + ((E + 2) & ~1u));
    __shared__ uint32_t rows_seen, last;
    __shared__ double part[8];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t e = threadIdx.x; e < E; e += 256) { hist[e] = 0; sums[e] = 0; }
    if (threadIdx.x == 0) rows_seen = 0;
    __syncthreads();
    for (uint32_t t = blockIdx.x * 8 + warp; t < T; t += gridDim.x * 8) {
        if (mask && !mask[t]) continue;
        const float *z = logits + t * pitch;
        float m = -CUDART_INF_F, s = 0;
        for (uint32_t e = lane; e < E; e += 32) m = fmaxf(m, z[e]);
        m = warp_max(m);
        for (uint32_t e = lane; e < E; e += 32) s += expf(z[e] - m);
        s = warp_sum(s);
        if (!(s < CUDART_INF_F)) { if (lane == 0) note_nonfinite(tune.status, t); }
        const float inv = 1.0f / s;
        for (uint32_t e = lane; e < E; e += 32) atomicAdd(&sums[e], (unsigned long long)__float2ll_rn(expf(z[e] - m) * inv * UNIT));
        for (uint32_t k = lane; k < K; k += 32) {
            const uint32_t e = ids[(uint64_t)t * K + k];
            if (e < E) atomicAdd(&hist[e], 1u); else atomicOr(tune.status, QW4SH_ERR_BOUNDS);
        }
        if (lane == 0) atomicAdd(&rows_seen, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < E; e += 256) {
        if (hist[e]) atomicAdd(&tune.counts[e], hist[e]);
        if (sums[e]) atomicAdd(&tune.prob_sums[e], sums[e]);
    }
    if (threadIdx.x == 0) atomicAdd(&tune.counts[E], rows_seen);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&tune.counts[E + 1], 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // the CTA that arrives last hands the sums out and leaves zeros for the next launch
    const uint32_t n = __ldcg(&tune.counts[E]);
    const bool bad = __ldcg(tune.status) & QW4SH_ERR_NONFINITE;
    double l = 0;
    for (uint32_t e = threadIdx.x; e < E; e += 256) {
        const uint32_t c = __ldcg(&tune.counts[e]);
        const double p = (double)__ldcg(&tune.prob_sums[e]) * (1.0 / 1099511627776.0);
        counts[e] = c;
        prob_sums[e] = bad ? CUDART_NAN_F : (float)p;
        l += (double)c * p;
        tune.counts[e] = 0; tune.prob_sums[e] = 0;
    }
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) part[warp] = l;
    __syncthreads();
    if (threadIdx.x == 0) {
        l = 0;
        for (int w = 0; w < 8; w++) l += part[w];
        *loss = bad ? CUDART_NAN_F : n ? (float)(l * (double)E / ((double)n * (double)n)) : 0.0f;
        counts[E] = n;
        tune.counts[E] = 0; tune.counts[E + 1] = 0;
    }
}

__global__ void __launch_bounds__(256) balance_backward_kernel(uint32_t E, uint32_t K, int norm, const float *__restrict__ logits, uint64_t pitch,
                                                               const uint32_t *__restrict__ ids, const uint8_t *__restrict__ mask, uint32_t T,
                                                               const uint32_t *__restrict__ counts, float loss_grad, const float *__restrict__ dw,
                                                               float *__restrict__ grad, uint64_t gpitch, uint32_t *status) {
    const uint32_t lane = threadIdx.x & 31, t = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= T) return;
    float *out = grad + t * gpitch;
    if (mask && !mask[t]) {
        for (uint32_t e = lane; e < E; e += 32) out[e] = 0;
        return;
    }
    const float *z = logits + t * pitch;
    const float n = (float)counts[E], scale = n > 0 ? loss_grad * (float)E / (n * n) : 0.0f;
    float m = -CUDART_INF_F, s = 0, f = 0;
    for (uint32_t e = lane; e < E; e += 32) m = fmaxf(m, z[e]);
    m = warp_max(m);
    for (uint32_t e = lane; e < E; e += 32) { const float p = expf(z[e] - m); s += p; f += p * ((float)counts[e] * scale); }
    s = warp_sum(s);
    f = warp_sum(f);
    if (!(s < CUDART_INF_F) && lane == 0) note_nonfinite(status, t);
    const float inv = 1.0f / s;
    f *= inv;
    const uint32_t *id = ids + (uint64_t)t * K;
    float top = -CUDART_INF_F, total = 0, mean = 0;       // over the chosen experts: largest logit, sum of weights, mean of dw
    if (dw) {
        for (uint32_t k = lane; k < K; k += 32) { if (id[k] < E) top = fmaxf(top, z[id[k]]); else atomicOr(status, QW4SH_ERR_BOUNDS); }
        top = warp_max(top);
        for (uint32_t k = lane; k < K; k += 32)
            if (id[k] < E) {
                const float w = norm ? expf(z[id[k]] - top) : expf(z[id[k]] - m) * inv;
                total += w;
                mean += w * dw[(uint64_t)t * K + k];
            }
        total = norm ? warp_sum(total) : 1.0f;
        mean = warp_sum(mean) / total;
    }
    const float shared = f + (norm ? 0.0f : mean);
    for (uint32_t e = lane; e < E; e += 32) out[e] = expf(z[e] - m) * inv * ((float)counts[e] * scale - shared);
    __syncwarp();
    if (dw)
        for (uint32_t k = 0; k < K; k++)                  // one after another: an id may be there twice
            if (lane == 0 && id[k] < E) {
                const float d = dw[(uint64_t)t * K + k];
                out[id[k]] += norm ? expf(z[id[k]] - top) / total * (d - mean) : expf(z[id[k]] - m) * inv * d;
            }
}

}  // namespace

extern "C" int qw4sh_balance_forward(const QW4ShTune *tune, uint32_t E, uint32_t K, const float *logits, size_t pitch, const uint32_t *ids,
                                     const uint8_t *mask, size_t tokens, uint32_t *counts, float *prob_sums, float *loss, void *stream) {
    const unsigned most = (unsigned)((tokens + 7) / 8);
    const unsigned grid = most < 1 ? 1 : most > 592 ? 592 : most;
    const size_t smem = (size_t)((E + 2) & ~1u) * 4 + (size_t)E * 8;
    if (smem > 48u * 1024u && cudaFuncSetAttribute(balance_forward_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return qw4sh_fail_text("balance_forward_kernel: shared memory");
    balance_forward_kernel<<<grid, 256, smem, (cudaStream_t)stream>>>(E, K, logits, pitch, ids, mask, (uint32_t)tokens, *tune, counts, prob_sums, loss);
    return qw4sh_note_launch("balance_forward_kernel");
}

extern "C" int qw4sh_balance_backward(const QW4ShTune *tune, uint32_t E, uint32_t K, int norm, const float *logits, size_t pitch, const uint32_t *ids,
                                      const uint8_t *mask, size_t tokens, const uint32_t *counts, float loss_grad, const float *weights_grad, float *grad,
                                      size_t grad_pitch, void *stream) {
    balance_backward_kernel<<<(unsigned)((tokens + 7) / 8), 256, 0, (cudaStream_t)stream>>>(E, K, norm, logits, pitch, ids, mask, (uint32_t)tokens, counts,
                                                                                          loss_grad, weights_grad, grad, grad_pitch, tune->status);
    return qw4sh_note_launch("balance_backward_kernel");
}
