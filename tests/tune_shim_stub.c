/* Stand-in for the CUDA shim, on host memory, under csrc/tune_host.c: a test of its argument checks needs no GPU.
 * A launch does nothing but count. */
#include <stdlib.h>
#include <string.h>

#include "../picoforge_b200/csrc/cuda_shim.h"

int stub_device, stub_launches, stub_fail_launch, stub_fail_malloc;
uint32_t stub_status[2] = {0, 0xffffffffu};             /* what the next sync finds */

size_t qw4sh_adapter_tiles(size_t tokens, uint32_t slots) { return tokens + slots; }
size_t qw4sh_adapter_rows(size_t tokens, uint32_t slots) { return tokens + slots; }
uint32_t qw4sh_adapter_rank(uint32_t rank) { return rank; }
int qw4sh_current_device(void) { return stub_device; }
int qw4sh_device_count(void) { return 2; }
const char *qw4sh_last_error(void) { return "stub"; }
void *qw4sh_malloc(size_t bytes) { return stub_fail_malloc ? NULL : malloc(bytes); }
void qw4sh_free(void *p) { free(p); }
void *qw4sh_host_alloc(size_t bytes) { return malloc(bytes); }
void qw4sh_host_free(void *p) { free(p); }
int qw4sh_memset_async(void *dst, int value, size_t bytes, void *stream) { (void)stream; memset(dst, value, bytes); return 0; }
int qw4sh_memcpy2d_async(void *dst, size_t dp, const void *src, size_t sp, size_t width, size_t rows, int to_device, void *stream) {
    (void)dp; (void)sp; (void)src; (void)rows; (void)to_device; (void)stream;
    memset(dst, 0, width);
    memcpy(dst, stub_status, 8);
    return 0;
}
int qw4sh_stream_sync(void *stream) { (void)stream; return 0; }
int qw4sh_current_stream(void **stream) { *stream = NULL; return 0; }
int qw4sh_balance_forward(const QW4ShTune *tune, uint32_t experts, uint32_t k, const float *logits, size_t pitch, const uint32_t *ids,
                          const uint8_t *mask, size_t tokens, uint32_t *counts, float *prob_sums, float *loss, void *stream) {
    (void)tune; (void)experts; (void)k; (void)logits; (void)pitch; (void)ids; (void)mask; (void)tokens; (void)counts; (void)prob_sums; (void)loss; (void)stream;
    stub_launches++;
    return stub_fail_launch;
}
int qw4sh_balance_backward(const QW4ShTune *tune, uint32_t experts, uint32_t k, int norm, const float *logits, size_t pitch, const uint32_t *ids,
                           const uint8_t *mask, size_t tokens, const uint32_t *counts, float loss_grad, const float *weights_grad, float *grad,
                           size_t grad_pitch, void *stream) {
    (void)tune; (void)experts; (void)k; (void)norm; (void)logits; (void)pitch; (void)ids; (void)mask; (void)tokens; (void)counts; (void)loss_grad;
    (void)weights_grad; (void)grad; (void)grad_pitch; (void)stream;
    stub_launches++;
    return stub_fail_launch;
}
int qw4sh_adapter_forward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                          const float *base, size_t base_pitch, float *y, size_t y_pitch, size_t tokens, void *stream) {
    (void)tune; (void)ad; (void)x; (void)x_pitch; (void)slots; (void)base; (void)base_pitch; (void)y; (void)y_pitch; (void)tokens; (void)stream;
    stub_launches++;
    return stub_fail_launch;
}
int qw4sh_adapter_backward(const QW4ShTune *tune, const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots,
                           const float *dy, size_t dy_pitch, const float *base, size_t base_pitch, float *dx, size_t dx_pitch,
                           float *da, float *db, size_t tokens, void *stream) {
    (void)tune; (void)ad; (void)x; (void)x_pitch; (void)slots; (void)dy; (void)dy_pitch; (void)base; (void)base_pitch; (void)dx; (void)dx_pitch;
    (void)da; (void)db; (void)tokens; (void)stream;
    stub_launches++;
    return stub_fail_launch;
}
