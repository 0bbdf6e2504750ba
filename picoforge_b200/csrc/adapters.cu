// Low-rank adapters of many requests beside a projection that they share, and their gradients (contract:
// include/qwen4_moe_b200.h; no counterpart in the reference).
//
//   h_t = A_s x_t            y_t  = base_t + scale_s B_s h_t
//   g_t = scale_s B_s^T dy_t  dx_t = base_t + A_s^T g_t     dA_s = sum_t g_t x_t^T     dB_s = scale_s sum_t dy_t h_t^T
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "cuda_shim.h"

extern "C" int qw4sh_note_launch(const char *name);

namespace {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// A slot's matrix read as [rank, width]: element (r, c) at r * sr + c * sc.
template <typename W> struct Mat { const W *p; uint64_t slot; uint64_t sr, sc; };

// h[t, r] = scale * sum_c w[slot][r, c] x[t, c]: one warp per (t, r).
template <typename W>
__global__ void __launch_bounds__(256) adapter_shrink_kernel(Mat<W> w, uint32_t S, uint32_t R, uint64_t width, const float *__restrict__ x, uint64_t pitch,
                                                             const uint32_t *__restrict__ slots, const float *__restrict__ scale, uint32_t T,
                                                             float *__restrict__ h, uint32_t *status) {
    const uint64_t at = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31, t = (uint32_t)(at / R), r = (uint32_t)(at % R);
    if (t >= T) return;
    const uint32_t s = slots[t];
    if (s >= S) {
        if (s != QW4CU_NO_ADAPTER && lane == 0) atomicOr(status, QW4SH_ERR_BOUNDS);
        return;
    }
    const W *m = w.p + s * w.slot + r * w.sr;
    const float *row = x + t * pitch;
    float sum = 0;
    for (uint64_t c = lane; c < width; c += 32) sum = fmaf(to_float(m[c * w.sc]), row[c], sum);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) h[at] = sum * (scale ? scale[s] : 1.0f);
}

// y[t, c] = base[t, c] + sum_r h[t, r] w[slot][r, c]
template <typename W>
__global__ void __launch_bounds__(256) adapter_expand_kernel(Mat<W> w, uint32_t S, uint32_t R, uint64_t width, const float *__restrict__ h,
                                                             const uint32_t *__restrict__ slots, uint32_t T, const float *base, uint64_t bpitch, float *y,
                                                             uint64_t ypitch) {
    const uint64_t c = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= width) return;
    for (uint32_t t = blockIdx.y; t < T; t += gridDim.y) {
        const uint32_t s = slots[t];
        float sum = 0;
        if (s < S) {
            const W *m = w.p + s * w.slot + c * w.sc;
            for (uint32_t r = 0; r < R; r++) sum = fmaf(to_float(m[r * w.sr]), h[(uint64_t)t * R + r], sum);
        }
        y[t * ypitch + c] = base ? base[t * bpitch + c] + sum : sum;
    }
}

// d[slot][r * sr + c * sc] = sum over the slot's tokens of h[t, r] x[t, c]
__global__ void __launch_bounds__(256) adapter_outer_kernel(float *__restrict__ d, uint64_t sr, uint64_t sc, uint32_t R, uint64_t width,
                                                            const float *__restrict__ h, const float *__restrict__ x, uint64_t pitch,
                                                            const uint32_t *__restrict__ slots, uint32_t T) {
    const uint64_t c = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t r = blockIdx.y, s = blockIdx.z;
    if (c >= width) return;
    float sum = 0;
    for (uint32_t t = 0; t < T; t++) if (slots[t] == s) sum = fmaf(h[(uint64_t)t * R + r], x[t * pitch + c], sum);
    d[s * ((uint64_t)R * width) + r * sr + c * sc] = sum;
}

template <typename W>
int shrink(Mat<W> w, const QW4CuAdapters *ad, uint64_t width, const float *x, size_t pitch, const uint32_t *slots, const float *scale, size_t T, float *h,
           uint32_t *status, cudaStream_t stream) {
    adapter_shrink_kernel<W><<<(unsigned)((T * ad->rank + 7) / 8), 256, 0, stream>>>(w, ad->slots, ad->rank, width, x, pitch, slots, scale, (uint32_t)T, h, status);
    return qw4sh_note_launch("adapter_shrink_kernel");
}
template <typename W>
int expand(Mat<W> w, const QW4CuAdapters *ad, uint64_t width, const float *h, const uint32_t *slots, size_t T, const float *base, size_t bpitch, float *y,
           size_t ypitch, cudaStream_t stream) {
    adapter_expand_kernel<W><<<dim3((unsigned)((width + 255) / 256), (unsigned)(T < 65535 ? T : 65535)), 256, 0, stream>>>(
        w, ad->slots, ad->rank, width, h, slots, (uint32_t)T, base, bpitch, y, ypitch);
    return qw4sh_note_launch("adapter_expand_kernel");
}

template <typename W> Mat<W> mat_a(const QW4CuAdapters *ad) { return {(const W *)ad->a, ad->rank * ad->k, ad->k, 1}; }
template <typename W> Mat<W> mat_b(const QW4CuAdapters *ad) { return {(const W *)ad->b, ad->rank * ad->n, 1, ad->rank}; }

template <typename W>
int forward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots, const float *base, size_t base_pitch,
            float *y, size_t y_pitch, size_t T, cudaStream_t stream) {
    if (const int rc = shrink<W>(mat_a<W>(ad), ad, ad->k, x, x_pitch, slots, ad->scale, T, tune->h, tune->status, stream)) return rc;
    return expand<W>(mat_b<W>(ad), ad, ad->n, tune->h, slots, T, base, base_pitch, y, y_pitch, stream);
}

template <typename W>
int backward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots, const float *dy, size_t dy_pitch,
             const float *base, size_t base_pitch, float *dx, size_t dx_pitch, float *da, float *db, size_t T, cudaStream_t stream) {
    int rc;
    if (T && (rc = shrink<W>(mat_b<W>(ad), ad, ad->n, dy, dy_pitch, slots, ad->scale, T, tune->g, tune->status, stream))) return rc;
    if (T && dx && (rc = expand<W>(mat_a<W>(ad), ad, ad->k, tune->g, slots, T, base, base_pitch, dx, dx_pitch, stream))) return rc;
    if (!da) return 0;
    if (T && (rc = shrink<W>(mat_a<W>(ad), ad, ad->k, x, x_pitch, slots, ad->scale, T, tune->h, tune->status, stream))) return rc;
    adapter_outer_kernel<<<dim3((unsigned)((ad->k + 255) / 256), ad->rank, ad->slots), 256, 0, stream>>>(da, ad->k, 1, ad->rank, ad->k, tune->g, x, x_pitch, slots, (uint32_t)T);
    if ((rc = qw4sh_note_launch("adapter_outer_kernel"))) return rc;
    adapter_outer_kernel<<<dim3((unsigned)((ad->n + 255) / 256), ad->rank, ad->slots), 256, 0, stream>>>(db, 1, ad->rank, ad->rank, ad->n, tune->h, dy, dy_pitch, slots, (uint32_t)T);
    return qw4sh_note_launch("adapter_outer_kernel");
}

}  // namespace

extern "C" int qw4sh_adapter_forward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                                     const float *base, size_t base_pitch, float *y, size_t y_pitch, size_t tokens, void *stream) {
    const auto run = ad->type == 0 ? forward<float> : ad->type == 1 ? forward<__half> : forward<__nv_bfloat16>;
    return run(tune, ad, x, x_pitch, slots, base, base_pitch, y, y_pitch, tokens, (cudaStream_t)stream);
}

extern "C" int qw4sh_adapter_backward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                                      const float *dy, size_t dy_pitch, const float *base, size_t base_pitch, float *dx, size_t dx_pitch,
                                      float *da, float *db, size_t tokens, void *stream) {
    const auto run = ad->type == 0 ? backward<float> : ad->type == 1 ? backward<__half> : backward<__nv_bfloat16>;
    return run(tune, ad, x, x_pitch, slots, dy, dy_pitch, base, base_pitch, dx, dx_pitch, da, db, tokens, (cudaStream_t)stream);
}
