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
extern "C" int qw4sh_allow_smem(const void *kernel, size_t smem);

namespace {

constexpr uint32_t THREADS = 256;

// Probability sums meet as 64-bit integers, whose sum has no order: multiples of 2^-40 in the first, and what is left of a share in multiples of
// 2^-82 in the second, so that an unlikely expert's sum keeps FP32's bits too.  Neither overflows: shares add up to no more than 2^20 tokens, and there
// are no more than that many of less than 2^42 each in the second.
constexpr uint32_t WHOLE = 40, REST = 82;
__host__ __device__ constexpr float two_to(uint32_t n) { return (float)(1ull << n / 2) * (float)(1ull << (n - n / 2)); }
// What v leaves of its multiples of 1 / unit (a power of two; nothing of a v of 2^24 of them or more), in multiples of 2^-REST.
__device__ __forceinline__ unsigned long long rest_of(float v, float unit) {
    return (unsigned long long)__float2ll_rn(fmaf(v, unit, -(float)__float2ll_rz(v * unit)) * (two_to(REST) / unit));
}

// By all lanes of a warp together: volatile, or the compiler may move it to where its result is used, which not every lane reaches.
__device__ __forceinline__ float warp_max(float v) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}
// exp(v - m) as 2^((v - m) log2 e): the difference and the product are rounded once each and the instruction is off by 2^-22 at most; -inf gives zero, and
// what has no softmax (a NaN, a +inf, nothing but -inf) a NaN.  Results below 2^-126 are zero: the form that keeps them takes four
// instructions, and these kernels are bound by instructions.  With expf 49152 x 512 takes 25.3 us instead of 23.3 and its gradient 46.3 instead of
// 44.5, and results are as far from 64 bits: sums 2e-8 to 8e-8 of their norm, gradients 5e-8 to 3.4e-7.
__device__ __forceinline__ float exp_of(float v, float m) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((v - m) * 1.4426950408889634f));
    return e;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Kernels here may begin before the launch ahead of them has ended: before the wait they read nothing, and what they read after it is no
// __restrict__ pointer to const, whose loads the compiler would be free to put before it.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// A row that has no softmax is noted with its number (the lowest is kept).
__device__ __noinline__ void note_nonfinite(uint32_t *status, uint32_t row) {
    atomicOr(status, QW4SH_ERR_NONFINITE);
    atomicMin(status + 1, row);
}

// A row of up to 32 * PER logits in a warp's registers: lane l holds columns (VEC) 4 l .. 4 l + 3 of every 128, or l of every 32; -inf
// behind the last one, which is a probability of zero.
template <int PER, bool VEC> struct Row {
    float v[PER];
    static __device__ __forceinline__ uint32_t column(int i, uint32_t lane) { return VEC ? 128 * (i / 4) + 4 * lane + i % 4 : 32 * i + lane; }
    __device__ __forceinline__ void load(const float *z, uint32_t E, uint32_t lane) {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                const uint32_t c = column(i, lane);
                const float4 u = c < E ? *(const float4 *)(z + c) : make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
                v[i] = u.x; v[(i + 1) % PER] = u.y; v[(i + 2) % PER] = u.z; v[(i + 3) % PER] = u.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = column(i, lane) < E ? z[column(i, lane)] : -CUDART_INF_F;
        }
    }
    // exp(v - m), their sum over the row
    __device__ __forceinline__ float exponentials(float &m) {
        m = v[0];
#pragma unroll
        for (int i = 1; i < PER; i++) m = fmaxf(m, v[i]);
        m = warp_max(m);
        float s = 0;
#pragma unroll
        for (int i = 0; i < PER; i++) { v[i] = exp_of(v[i], m); s += v[i]; }
        return warp_sum(s);
    }
};

__device__ __forceinline__ void add_rest(const QW4ShTune &tune, uint32_t e, unsigned long long rest) {
    if (rest) { atomicAdd(&tune.prob_rests[e], rest); tune.status[3] = 1; }
}

// The end of the forward pass: the CTA that arrives last hands the sums out and leaves zeros for the next launch.
__device__ __forceinline__ void balance_finish(uint32_t E, const QW4ShTune &tune, uint32_t *counts, float *prob_sums, float *loss) {
    __shared__ uint32_t last;
    __shared__ double part[THREADS / 32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&tune.counts[E + 1], 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    const uint32_t n = __ldcg(&tune.counts[E]);
    const bool bad = __ldcg(tune.status + 2), rests = __ldcg(tune.status + 3);
    double l = 0;
    for (uint32_t e = threadIdx.x; e < E; e += THREADS) {
        const uint32_t c = __ldcg(&tune.counts[e]);
        double p = (double)__ldcg(&tune.prob_sums[e]) * (1.0 / (double)two_to(WHOLE));
        if (rests) { p += (double)__ldcg(&tune.prob_rests[e]) * (1.0 / (double)two_to(REST)); tune.prob_rests[e] = 0; }
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
        for (uint32_t w = 0; w < THREADS / 32; w++) l += part[w];
        *loss = bad ? CUDART_NAN_F : n ? (float)(l * (double)E / ((double)n * (double)n)) : 0.0f;
        counts[E] = n;
        tune.counts[E] = 0; tune.counts[E + 1] = 0; tune.status[2] = tune.status[3] = 0;
    }
}

// A warp to a row, the next row on its way while one is summed; every lane adds up its columns in registers over the rows of its warp,
// the warps of a CTA add theirs in shared memory, the CTAs as integers.
template <int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) balance_forward_kernel(uint32_t E, uint32_t K, const float *logits, uint64_t pitch,
                                                                  const uint32_t *ids, const uint8_t *mask, uint32_t T,
                                                                  const __grid_constant__ QW4ShTune tune, uint32_t *__restrict__ counts,
                                                                  float *__restrict__ prob_sums, float *__restrict__ loss) {
    constexpr uint32_t WARPS = THREADS / 32, COLS = 32 * PER;
    extern __shared__ float sums[];                          // [WARPS][COLS], then counts [COLS]
    uint32_t *hist = (uint32_t *)(sums + WARPS * COLS);
    __shared__ uint32_t rows_seen;
    using R = Row<PER, VEC>;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, step = gridDim.x * WARPS;
    for (uint32_t e = threadIdx.x; e < COLS; e += THREADS) hist[e] = 0;
    if (threadIdx.x == 0) rows_seen = 0;
    grid_wait();
    __syncthreads();
    uint32_t t = blockIdx.x * WARPS + warp, seen = 0;
    float acc[PER] = {};
    R next;
    bool there = t < T && (!mask || mask[t]);
    if (there) next.load(logits + t * pitch, E, lane);
    uint32_t id = there && lane < K ? ids[(uint64_t)t * K + lane] : 0;
    for (; t < T; t += step) {
        R row = next;
        const bool now = there;
        const uint32_t now_id = id, t_next = t + step;
        there = t_next < T && (!mask || mask[t_next]);
        if (there) {
            next.load(logits + t_next * pitch, E, lane);
            id = lane < K ? ids[(uint64_t)t_next * K + lane] : 0;
        }
        if (!now) continue;
        float m;
        const float s = row.exponentials(m);
        if (!(s < CUDART_INF_F)) { if (lane == 0) { note_nonfinite(tune.status, t); tune.status[2] = 1; } }
        const float inv = 1.0f / s;
#pragma unroll
        for (int i = 0; i < PER; i++) acc[i] = fmaf(row.v[i], inv, acc[i]);
        for (uint32_t k = lane; k < K; k += 32) {
            const uint32_t e = k < 32 ? now_id : ids[(uint64_t)t * K + k];
            if (e < E) atomicAdd(&hist[e], 1u); else atomicOr(tune.status, QW4SH_ERR_BOUNDS);
        }
        seen++;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) sums[warp * COLS + R::column(i, lane)] = acc[i];
    if (lane == 0 && seen) atomicAdd(&rows_seen, seen);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < E; e += THREADS) {
        float sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; w++) sum += sums[w * COLS + e];
        const unsigned long long whole = (unsigned long long)__float2ll_rz(sum * two_to(WHOLE));
        if (whole) atomicAdd(&tune.prob_sums[e], whole);
        if (sum < two_to(24) / two_to(WHOLE)) {
            add_rest(tune, e, rest_of(sum, two_to(WHOLE)));
        }
        if (hist[e]) atomicAdd(&tune.counts[e], hist[e]);
    }
    if (threadIdx.x == 0 && rows_seen) atomicAdd(&tune.counts[E], rows_seen);
    balance_finish(E, tune, counts, prob_sums, loss);
}

// More experts than fit a warp's registers: a warp to a row, three passes over it (the later ones out of L1), every probability
// added to the CTA's sums as an integer, in multiples of 2^-unit: as fine as the CTA's rows leave room for.  What that leaves of a probability goes past
// them, so that it takes no shared memory (two sums to an expert there: 8192 x 4096 157 us instead of 132).
__global__ void __launch_bounds__(THREADS) balance_forward_wide_kernel(uint32_t E, uint32_t K, const float *logits, uint64_t pitch,
                                                                       const uint32_t *ids, const uint8_t *mask, uint32_t T,
                                                                       const __grid_constant__ QW4ShTune tune, uint32_t unit, uint32_t *__restrict__ counts,
                                                                       float *__restrict__ prob_sums, float *__restrict__ loss) {
    extern __shared__ uint32_t shared_words[];               // [E] counts, [E] sums as 64-bit integers
    uint32_t *hist = shared_words;
    unsigned long long *sums = (unsigned long long *)(hist + ((E + 1) & ~1u));
    __shared__ uint32_t rows_seen;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float scale = two_to(unit), few_bits = two_to(24) / scale;
    for (uint32_t e = threadIdx.x; e < E; e += THREADS) { hist[e] = 0; sums[e] = 0; }
    if (threadIdx.x == 0) rows_seen = 0;
    grid_wait();
    __syncthreads();
    for (uint32_t t = blockIdx.x * (THREADS / 32) + warp; t < T; t += gridDim.x * (THREADS / 32)) {
        if (mask && !mask[t]) continue;
        const float *z = logits + t * pitch;
        float m = -CUDART_INF_F, s = 0;
        for (uint32_t e = lane; e < E; e += 32) m = fmaxf(m, z[e]);
        m = warp_max(m);
        for (uint32_t e = lane; e < E; e += 32) s += expf(z[e] - m);
        s = warp_sum(s);
        if (!(s < CUDART_INF_F)) { if (lane == 0) { note_nonfinite(tune.status, t); tune.status[2] = 1; } }
        const float inv = 1.0f / s;
        bool small = false;
        for (uint32_t e = lane; e < E; e += 32) {
            const float p = expf(z[e] - m) * inv;
            small |= p < few_bits && p > 0;
            atomicAdd(&sums[e], (unsigned long long)__float2ll_rz(p * scale));
        }
        if (small)                                           // a pass of its own: inside the other one it cost that a tenth
            for (uint32_t e = lane; e < E; e += 32) {
                const float p = expf(z[e] - m) * inv;
                if (p < few_bits) add_rest(tune, e, rest_of(p, scale));
            }
        for (uint32_t k = lane; k < K; k += 32) {
            const uint32_t e = ids[(uint64_t)t * K + k];
            if (e < E) atomicAdd(&hist[e], 1u); else atomicOr(tune.status, QW4SH_ERR_BOUNDS);
        }
        if (lane == 0) atomicAdd(&rows_seen, 1u);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < E; e += THREADS) {
        if (hist[e]) atomicAdd(&tune.counts[e], hist[e]);
        const unsigned long long whole = sums[e] >> (unit - WHOLE), rest = sums[e] - (whole << (unit - WHOLE)) << (REST - unit);
        if (whole) atomicAdd(&tune.prob_sums[e], whole);
        add_rest(tune, e, rest);
    }
    if (threadIdx.x == 0 && rows_seen) atomicAdd(&tune.counts[E], rows_seen);
    balance_finish(E, tune, counts, prob_sums, loss);
}

// A warp to a row.  The share of the route weights is worked out by a lane per chosen expert and laid over the row behind the rest.
template <int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) balance_backward_kernel(uint32_t E, uint32_t K, int norm, const float *logits, uint64_t pitch,
                                                                   const uint32_t *ids, const uint8_t *mask, uint32_t T,
                                                                   const uint32_t *counts, float loss_grad, const float *dw,
                                                                   float *__restrict__ grad, uint64_t gpitch, uint32_t *status) {
    constexpr uint32_t WARPS = THREADS / 32;
    using R = Row<PER, VEC>;
    const uint32_t lane = threadIdx.x & 31, step = gridDim.x * WARPS;
    uint32_t t = blockIdx.x * WARPS + (threadIdx.x >> 5);
    grid_wait();
    const float n = (float)counts[E], scale = n > 0 ? loss_grad * (float)E / (n * n) : 0.0f;
    float f[PER];                                            // d loss / d p of the lane's columns
#pragma unroll
    for (int i = 0; i < PER; i++) { const uint32_t c = R::column(i, lane); f[i] = c < E ? (float)counts[c] * scale : 0.0f; }
    const bool chosen = dw && lane < K;
    R next;
    uint32_t id = 0;
    float d = 0, zc = 0;
    auto fetch = [&](uint32_t row) -> bool {
        if (row >= T || (mask && !mask[row])) return false;
        next.load(logits + row * pitch, E, lane);
        if (chosen) { id = ids[(uint64_t)row * K + lane]; d = dw[(uint64_t)row * K + lane]; }
        return true;
    };
    bool there = fetch(t);
    for (; t < T; t += step) {
        R row = next;
        const bool now = there;
        const uint32_t my_id = id;
        const float my_d = d;
        float *out = grad + t * gpitch;
        const bool in = chosen && now && my_id < E;
        float f_mine = 0;
        if (in) { zc = logits[t * pitch + my_id]; f_mine = (float)counts[my_id] * scale; }
        there = fetch(t + step);
        float values[PER], total = 0, shared = 0, p_mine = 0;       // total: the route weights' share
        uint32_t same = 0;
        if (now) {
            float m;
            const float s = row.exponentials(m);
            if (!(s < CUDART_INF_F) && lane == 0) note_nonfinite(status, t);
            const float inv = 1.0f / s;
            float sum = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) sum = fmaf(row.v[i], f[i], sum);
            shared = warp_sum(sum) * inv;
            if (dw) {
                if (chosen && my_id >= E) atomicOr(status, QW4SH_ERR_BOUNDS);
                p_mine = in ? exp_of(zc, m) * inv : 0.0f;
                if (norm) {
                    const float top = warp_max(in ? zc : -CUDART_INF_F);
                    const float w = in ? expf(zc - top) : 0.0f;
                    const float weight = w / warp_sum(w);
                    const float mean = warp_sum(in ? weight * my_d : 0.0f);
                    total = in ? weight * (my_d - mean) : 0.0f;
                } else {
                    const float mean = warp_sum(in ? p_mine * my_d : 0.0f);
                    total = in ? p_mine * my_d : 0.0f;
                    shared += mean;
                }
                same = __match_any_sync(0xffffffffu, in ? my_id : 0x80000000u | lane);
            }
            const float off = shared * inv;
#pragma unroll
            for (int i = 0; i < PER; i++) values[i] = row.v[i] * fmaf(f[i], inv, -off);
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) values[i] = 0;
        }
        if (VEC && gpitch % 4 == 0 && ((uintptr_t)grad & 15) == 0) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                const uint32_t c = R::column(i, lane);
                if (c < E) *(float4 *)(out + c) = make_float4(values[i], values[(i + 1) % PER], values[(i + 2) % PER], values[(i + 3) % PER]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; i++) if (R::column(i, lane) < E) out[R::column(i, lane)] = values[i];
        }
        if (now && dw) {
            if (__any_sync(0xffffffffu, in && (same & (same - 1)))) {                // an expert that is there twice gets the sum, in the slots' order
                float all = 0;
                for (uint32_t k = 0; k < 32; k++) { const float u = __shfl_sync(0xffffffffu, total, k); if (same >> k & 1) all += u; }
                total = all;
            }
            __syncwarp();
            if (in) out[my_id] = p_mine * (f_mine - shared) + total;
        }
    }
}

// More experts than fit a warp's registers, or more chosen ones than lanes.
__global__ void __launch_bounds__(THREADS) balance_backward_wide_kernel(uint32_t E, uint32_t K, int norm, const float *logits, uint64_t pitch,
                                                                        const uint32_t *ids, const uint8_t *mask, uint32_t T,
                                                                        const uint32_t *counts, float loss_grad, const float *dw,
                                                                        float *__restrict__ grad, uint64_t gpitch, uint32_t *status) {
    const uint32_t lane = threadIdx.x & 31, t = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    grid_wait();
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

namespace {

constexpr unsigned SMS = 148;
template <typename... P, typename... A>
int launch(void (*kernel)(P...), const char *name, unsigned grid, size_t smem, void *stream, A... args) {
    if (smem > 40u * 1024u && qw4sh_allow_smem((const void *)kernel, smem)) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization; attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    return qw4sh_note_launch(name);
}
// CTAs for T rows of a warp each: no more than `per_sm` to an SM, which then take the rows in turn.
unsigned grid_of(size_t T, unsigned per_sm) {
    const size_t most = (T + THREADS / 32 - 1) / (THREADS / 32);
    return (unsigned)(most < 1 ? 1 : most < per_sm * SMS ? most : per_sm * SMS);
}
bool vectors(const float *p, size_t pitch, uint32_t E) { return E % 4 == 0 && pitch % 4 == 0 && ((uintptr_t)p & 15) == 0; }

}  // namespace

// The narrowest row that holds E columns; in runs of four where rows lie on boundaries of four.
#define BY_ROW(kernel, run) \
    (E <= 64 ? run((kernel<2, false>), 2) : E <= 128 ? (vec ? run((kernel<4, true>), 4) : run((kernel<4, false>), 4)) : \
     E <= 256 ? (vec ? run((kernel<8, true>), 8) : run((kernel<8, false>), 8)) : E <= 512 ? (vec ? run((kernel<16, true>), 16) : run((kernel<16, false>), 16)) : \
     (vec ? run((kernel<32, true>), 32) : run((kernel<32, false>), 32)))

extern "C" int qw4sh_balance_forward(const QW4ShTune *tune, uint32_t E, uint32_t K, const float *logits, size_t pitch, const uint32_t *ids,
                                     const uint8_t *mask, size_t tokens, uint32_t *counts, float *prob_sums, float *loss, void *stream) {
    const bool vec = vectors(logits, pitch, E);
#define RUN(kernel, per) launch(kernel, "balance_forward_kernel", grid_of(tokens, 3), (THREADS / 32 + 1) * 32 * per * 4, stream, E, K, logits, pitch, ids, mask, \
                                (uint32_t)tokens, *tune, counts, prob_sums, loss)
    if (E <= 1024) return BY_ROW(balance_forward_kernel, RUN);
#undef RUN
    const unsigned grid = grid_of(tokens, 4);
    const size_t rows = (tokens + grid * (THREADS / 32) - 1) / (grid * (THREADS / 32)) * (THREADS / 32);                       // of a CTA
    uint32_t unit = 62;
    while (rows > 1ull << (62 - unit)) unit--;
    return launch(balance_forward_wide_kernel, "balance_forward_wide_kernel", grid, (size_t)((E + 1) & ~1u) * 4 + (size_t)E * 8, stream, E, K, logits,
                  pitch, ids, mask, (uint32_t)tokens, *tune, unit, counts, prob_sums, loss);
}

extern "C" int qw4sh_balance_backward(const QW4ShTune *tune, uint32_t E, uint32_t K, int norm, const float *logits, size_t pitch, const uint32_t *ids,
                                      const uint8_t *mask, size_t tokens, const uint32_t *counts, float loss_grad, const float *weights_grad, float *grad,
                                      size_t grad_pitch, void *stream) {
    const bool vec = vectors(logits, pitch, E);
#define RUN(kernel, per) launch(kernel, "balance_backward_kernel", grid_of(tokens, 2), 0, stream, E, K, norm, logits, pitch, ids, mask, (uint32_t)tokens, counts, \
                                loss_grad, weights_grad, grad, grad_pitch, tune->status)
    if (E <= 1024 && K <= 32) return BY_ROW(balance_backward_kernel, RUN);
#undef RUN
    return launch(balance_backward_wide_kernel, "balance_backward_wide_kernel", (unsigned)((tokens + THREADS / 32 - 1) / (THREADS / 32)), 0, stream, E, K, norm, logits,
                  pitch, ids, mask, (uint32_t)tokens, counts, loss_grad, weights_grad, grad, grad_pitch, tune->status);
}
