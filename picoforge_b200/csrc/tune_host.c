/* Host side of the operators that adapt and train a layer: workspaces, argument checks, the latch.  The kernels are in
 * adapters.cu and balance.cu; the contract is in include/qwen4_moe_b200.h. */
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/qwen4_moe_b200.h"
#include "cuda_shim.h"

struct QW4CuTuneWork {
    QW4CuTuneLimits limits;
    int device;
    bool failed;
    size_t device_bytes, clear_bytes;     /* what has to be zero between launches lies in front */
    unsigned char *block;                 /* one device allocation carved into d.* */
    uint32_t status_host[4];
    QW4ShTune d;
};

static Qwen4Status answer(Qwen4Error *err, Qwen4Status code, const char *detail) {
    if (err) {
        memset(err, 0, sizeof *err);
        err->code = code;
        if (code != QW4_OK) {
            snprintf(err->subject, sizeof err->subject, "tune");
            snprintf(err->detail, sizeof err->detail, "%s", detail);
        }
    }
    return code;
}
static Qwen4Status cuda_answer(Qwen4Error *err, const char *what) {
    char text[256];
    snprintf(text, sizeof text, "%s: %.180s", what, qw4sh_last_error());
    return answer(err, QW4_GPU_ERROR, text);
}

/* ---- workspace -------------------------------------------------------------------------- */
static size_t take(size_t *at, size_t bytes) {
    const size_t here = *at;
    *at += (bytes + 255) & ~(size_t)255;
    return here;
}
/* The status words: no error, no bad row yet. */
static int status_clear(QW4CuTuneWork *w, void *stream) {
    return qw4sh_memset_async(w->d.status, 0, 4, stream) || qw4sh_memset_async(w->d.status + 1, 0xff, 4, stream);
}

Qwen4Status qw4cu_tune_work_create(const QW4CuTuneLimits *limits, QW4CuTuneWork **out, Qwen4Error *err) {
    if (out) *out = NULL;
    if (!limits || !out) return answer(err, QW4_INVALID_ARGUMENT, "null limits or output");
    const QW4CuTuneLimits l = *limits;
    if (!l.tokens || l.tokens > QW4CU_TUNE_MAX_TOKENS) return answer(err, QW4_RANGE, "tokens outside 1 .. 2^20");
    if (!l.slots && !l.experts) return answer(err, QW4_RANGE, "neither adapters nor experts");
    if (l.slots > QW4CU_TUNE_MAX_SLOTS || (l.slots && (!l.rank || l.rank > QW4CU_TUNE_MAX_RANK)))
        return answer(err, QW4_RANGE, "adapter slots beyond 1024 or rank outside 1 .. 128");
    if (l.experts > QW4CU_TUNE_MAX_EXPERTS) return answer(err, QW4_RANGE, "experts beyond 4096");
    QW4CuTuneWork *w = calloc(1, sizeof *w);
    if (!w) return answer(err, QW4_OOM, "workspace");
    w->limits = l;
    w->device = qw4sh_current_device();
    size_t at = 0;
    const size_t status = take(&at, 16), sums = take(&at, (size_t)l.experts * 8), counts = take(&at, ((size_t)l.experts + 2) * 4);
    const size_t rests = take(&at, (size_t)l.experts * 8);
    w->clear_bytes = at;
    const bool adapters = l.slots != 0;
    const size_t places = adapters ? qw4sh_adapter_rows(l.tokens, l.slots) : 0;
    const size_t order = take(&at, places * 4), offsets = take(&at, adapters ? ((size_t)l.slots + 1) * 8 : 0);
    const size_t tiles = take(&at, adapters ? qw4sh_adapter_tiles(l.tokens, l.slots) * 16 : 0), n_tiles = take(&at, 4);
    const size_t rows = adapters ? 3 * places * qw4sh_adapter_rank(l.rank) * 2 : 0, h = take(&at, rows), g = take(&at, rows);
    w->device_bytes = at;
    w->block = qw4sh_malloc(at);
    void *stream = NULL;
    if (!w->block || qw4sh_current_stream(&stream)) {
        const bool oom = qw4sh_device_count() > 0 && w->device >= 0;
        Qwen4Status st = cuda_answer(err, "workspace");
        if (oom && !w->block) { st = QW4_OOM; if (err) err->code = st; }
        qw4cu_tune_work_destroy(w);
        return st;
    }
    w->d.status = (uint32_t *)(w->block + status);
    w->d.prob_sums = (unsigned long long *)(w->block + sums);
    w->d.prob_rests = (unsigned long long *)(w->block + rests);
    w->d.counts = (uint32_t *)(w->block + counts);
    w->d.order = (uint32_t *)(w->block + order);
    w->d.offsets = (uint32_t *)(w->block + offsets);
    w->d.tiles = w->block + tiles;
    w->d.n_tiles = (uint32_t *)(w->block + n_tiles);
    w->d.h = w->block + h;
    w->d.g = w->block + g;
    if (qw4sh_memset_async(w->block, 0, w->clear_bytes, stream) || status_clear(w, stream) || qw4sh_stream_sync(stream)) {
        const Qwen4Status st = cuda_answer(err, "workspace clear");
        qw4cu_tune_work_destroy(w);
        return st;
    }
    *out = w;
    return answer(err, QW4_OK, "");
}
void qw4cu_tune_work_destroy(QW4CuTuneWork *w) {
    if (!w) return;
    qw4sh_free(w->block);
    free(w);
}
size_t qw4cu_tune_work_device_bytes(const QW4CuTuneWork *w) { return w ? w->device_bytes : 0; }

static Qwen4Status stream_of(const QW4CuTuneWork *w, void **stream, Qwen4Error *err) {
    if (qw4sh_current_device() != w->device) return answer(err, QW4_OWNER, "the workspace belongs to another device than the current one");
    return qw4sh_current_stream(stream) ? cuda_answer(err, "stream") : QW4_OK;
}

Qwen4Status qw4cu_tune_work_sync(QW4CuTuneWork *w, Qwen4Error *err) {
    if (!w) return answer(err, QW4_INVALID_ARGUMENT, "null workspace");
    void *stream;
    const Qwen4Status st = stream_of(w, &stream, err);
    if (st != QW4_OK) return st;
    if (qw4sh_memcpy2d_async(w->status_host, 16, w->d.status, 16, 16, 1, 0, stream) || qw4sh_stream_sync(stream)) {
        w->failed = true;
        return cuda_answer(err, "stream synchronize");
    }
    const uint32_t bits = w->status_host[0], row = w->status_host[1];
    if (!bits) return answer(err, QW4_OK, "");
    w->failed = true;
    if (bits & QW4SH_ERR_STATE) return answer(err, QW4_GPU_ERROR, "device state error");
    if (bits & QW4SH_ERR_BOUNDS) return answer(err, QW4_RANGE, "adapter slot or expert id out of range");
    const Qwen4Status bad = answer(err, QW4_NONFINITE, "a row of logits has no softmax");
    if (err && row != UINT32_MAX) err->row = row;
    return bad;
}
Qwen4Status qw4cu_tune_work_reset(QW4CuTuneWork *w, Qwen4Error *err) {
    if (!w) return answer(err, QW4_INVALID_ARGUMENT, "null workspace");
    void *stream;
    const Qwen4Status st = stream_of(w, &stream, err);
    if (st != QW4_OK) return st;
    if (qw4sh_memset_async(w->block, 0, w->clear_bytes, stream) || status_clear(w, stream) || qw4sh_stream_sync(stream))
        return cuda_answer(err, "workspace clear");
    w->failed = false;
    return answer(err, QW4_OK, "");
}

/* ---- arguments ---------------------------------------------------------------------------- */
typedef struct { uintptr_t first, end; size_t rows, row, pitch; } Bytes;

/* rows x row_bytes bytes, `pitch` bytes apart; what is wrong with it, or NULL. */
static const char *view(const void *p, size_t rows, size_t row_bytes, size_t pitch, size_t align, Bytes *out, Qwen4Status *code) {
    *code = QW4_INVALID_ARGUMENT;
    if (!p) return "null device view";
    if ((uintptr_t)p % align) return "device view not aligned to its elements";
    *code = QW4_STRIDE;
    if (pitch < row_bytes || pitch % align) return "row pitch shorter than a row or not a multiple of the element";
    *code = QW4_OVERFLOW;
    if (rows && pitch > (SIZE_MAX / 2 - row_bytes) / rows) return "extent overflow";
    const size_t bytes = rows ? (rows - 1) * pitch + row_bytes : 0;
    if ((uintptr_t)p + bytes < (uintptr_t)p) return "address overflow";
    *out = (Bytes){(uintptr_t)p, (uintptr_t)p + bytes, rows, row_bytes, pitch};
    return NULL;
}
/* Whether two views share a byte.  Rows of one pitch can lie between one another (columns of a wider buffer); of different pitches they are
 * taken to meet where the address ranges do. */
static bool meet(Bytes a, Bytes b) {
    if (a.first >= b.end || b.first >= a.end) return false;
    if (a.first > b.first) { const Bytes c = a; a = b; b = c; }
    if (a.rows == 1) return true;                                    /* b begins inside the only row */
    if (b.rows > 1 && a.pitch != b.pitch) return true;
    const size_t into = (b.first - a.first) % a.pitch;               /* b begins in a row of a, or behind one and reaches the next */
    return into < a.row || into + b.row > a.pitch;
}
#define VIEW(p, rows, row_bytes, pitch, align, out) do { Qwen4Status code_; const char *bad_ = view((p), (rows), (row_bytes), (pitch), (align), (out), &code_); \
    if (bad_) return answer(err, code_, bad_); } while (0)
#define TRY(call) do { const Qwen4Status st_ = (call); if (st_ != QW4_OK) return st_; } while (0)

static Qwen4Status usable(const QW4CuTuneWork *w, size_t tokens, void **stream, Qwen4Error *err) {
    if (!w) return answer(err, QW4_INVALID_ARGUMENT, "null workspace");
    if (w->failed) return answer(err, QW4_BAD_STATE, "failed workspace; reset required");
    if (tokens > w->limits.tokens) return answer(err, QW4_CAPACITY, "batch exceeds the workspace's tokens");
    return stream_of(w, stream, err);
}
/* Every written view apart from every other view, except that written[same_w] may be read[same_r] (the same rows). */
static Qwen4Status apart(const Bytes *written, size_t nw, const Bytes *read, size_t nr, size_t same_w, size_t same_r, Qwen4Error *err) {
    for (size_t i = 0; i < nw; i++) {
        for (size_t j = 0; j < nr; j++)
            if (meet(written[i], read[j]) && !(i == same_w && j == same_r)) return answer(err, QW4_INVALID_ARGUMENT, "an output overlaps an input");
        for (size_t j = i + 1; j < nw; j++) if (meet(written[i], written[j])) return answer(err, QW4_INVALID_ARGUMENT, "two outputs overlap");
    }
    return QW4_OK;
}

enum { MAX_DIM = 1u << 20 };
static Qwen4Status check_adapters(const QW4CuAdapters *ad, const QW4CuTuneWork *w, Bytes *a, Bytes *b, Bytes *scale, Qwen4Error *err) {
    if (!ad) return answer(err, QW4_INVALID_ARGUMENT, "null adapters");
    if (!ad->k || !ad->n || ad->k > MAX_DIM || ad->n > MAX_DIM) return answer(err, QW4_SHAPE, "projection dimensions outside 1 .. 2^20");
    if (!ad->slots || !ad->rank) return answer(err, QW4_SHAPE, "adapters of no slot or rank zero");
    if (ad->slots > w->limits.slots || ad->rank > w->limits.rank) return answer(err, QW4_CAPACITY, "adapter slots or rank beyond the workspace's");
    if (ad->type != 0 && ad->type != 1 && ad->type != 30) return answer(err, QW4_TYPE, "adapters are F32, F16 or BF16");
    const size_t e = ad->type == 0 ? 4 : 2;
    VIEW(ad->a, ad->slots, ad->rank * ad->k * e, ad->rank * ad->k * e, e, a);
    VIEW(ad->b, ad->slots, ad->rank * ad->n * e, ad->rank * ad->n * e, e, b);
    *scale = (Bytes){0};
    if (ad->scale) VIEW(ad->scale, 1, ad->slots * 4, ad->slots * 4, 4, scale);
    return QW4_OK;
}

Qwen4Status qw4tune_beside(const QW4CuAdapters *ad, size_t k, size_t n, const uint32_t *slots, size_t tokens, QW4CuTuneWork *w,
                           const QW4ShTune **tune, Qwen4Error *err) {
    void *stream;
    Bytes at;
    TRY(usable(w, tokens, &stream, err));
    TRY(check_adapters(ad, w, &at, &at, &at, err));
    if (ad->k != k || ad->n != n) return answer(err, QW4_SHAPE, "adapters of another projection");
    if (tokens) VIEW(slots, 1, tokens * 4, tokens * 4, 4, &at);
    *tune = &w->d;
    return QW4_OK;
}

static Bytes dense(const void *p, size_t bytes) { return p ? (Bytes){(uintptr_t)p, (uintptr_t)p + bytes, 1, bytes, bytes} : (Bytes){0}; }
Qwen4Status qw4tune_logits_out(const float *logits, size_t tokens, size_t hidden, size_t experts, size_t top_k, const float *x, const float *y,
                               const uint32_t *ids, const float *weights, const QW4CuAdapters *ad, const uint32_t *slots, Qwen4Error *err) {
    if (!logits) return answer(err, QW4_OK, "");
    Bytes out, others[8] = {dense(x, tokens * hidden * 4), dense(y, tokens * hidden * 4), dense(ids, tokens * top_k * 4), dense(weights, tokens * top_k * 4)};
    if (ad) {
        const size_t e = ad->type == 0 ? 4 : 2;
        others[4] = dense(slots, tokens * 4);
        others[5] = dense(ad->a, ad->slots * ad->rank * ad->k * e);
        others[6] = dense(ad->b, ad->slots * ad->rank * ad->n * e);
        others[7] = dense(ad->scale, ad->slots * 4);
    }
    VIEW(logits, 1, tokens * experts * 4, tokens * experts * 4, 4, &out);
    return apart(&out, 1, others, 8, 1, 8, err) == QW4_OK ? answer(err, QW4_OK, "") : answer(err, QW4_INVALID_ARGUMENT, "the logits overlap another argument");
}

Qwen4Status qw4cu_adapter_forward_device(const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots, const float *base,
                                         size_t base_pitch, float *y, size_t y_pitch, size_t tokens, QW4CuTuneWork *w, Qwen4Error *err) {
    void *stream;
    TRY(usable(w, tokens, &stream, err));
    Bytes read[6] = {{0}}, out;
    TRY(check_adapters(ad, w, &read[0], &read[1], &read[2], err));
    if (!tokens) return answer(err, QW4_OK, "");
    VIEW(x, tokens, ad->k * 4, x_pitch, 4, &read[3]);
    VIEW(slots, 1, tokens * 4, tokens * 4, 4, &read[4]);
    VIEW(y, tokens, ad->n * 4, y_pitch, 4, &out);
    if (base) VIEW(base, tokens, ad->n * 4, base_pitch, 4, &read[5]);
    TRY(apart(&out, 1, read, 6, 0, base == y && base_pitch == y_pitch ? 5 : 6, err));
    if (qw4sh_adapter_forward(&w->d, ad, x, x_pitch / 4, slots, base, base_pitch / 4, y, y_pitch / 4, tokens, stream)) return cuda_answer(err, "adapter launch");
    return answer(err, QW4_OK, "");
}

Qwen4Status qw4cu_adapter_backward_device(const QW4CuAdapters *ad, const float *x, size_t x_pitch, const uint32_t *slots, const float *dy,
                                          size_t dy_pitch, const float *base, size_t base_pitch, float *dx, size_t dx_pitch, float *da, float *db,
                                          size_t tokens, QW4CuTuneWork *w, Qwen4Error *err) {
    void *stream;
    TRY(usable(w, tokens, &stream, err));
    Bytes read[7] = {{0}}, out[3] = {{0}};
    TRY(check_adapters(ad, w, &read[0], &read[1], &read[2], err));
    if (!da != !db) return answer(err, QW4_INVALID_ARGUMENT, "da and db are given together");
    if (!dx && !da) return answer(err, QW4_INVALID_ARGUMENT, "no gradient asked for");
    if (tokens) {
        VIEW(slots, 1, tokens * 4, tokens * 4, 4, &read[3]);
        VIEW(dy, tokens, ad->n * 4, dy_pitch, 4, &read[4]);
        if (da) VIEW(x, tokens, ad->k * 4, x_pitch, 4, &read[5]);
        if (dx) VIEW(dx, tokens, ad->k * 4, dx_pitch, 4, &out[0]);
        if (dx && base) VIEW(base, tokens, ad->k * 4, base_pitch, 4, &read[6]);
    }
    if (da) {
        VIEW(da, ad->slots, ad->rank * ad->k * 4, ad->rank * ad->k * 4, 4, &out[1]);
        VIEW(db, ad->slots, ad->rank * ad->n * 4, ad->rank * ad->n * 4, 4, &out[2]);
    }
    TRY(apart(out, 3, read, 7, 0, base == dx && base_pitch == dx_pitch ? 6 : 7, err));
    if (qw4sh_adapter_backward(&w->d, ad, x, x_pitch / 4, slots, dy, dy_pitch / 4, base, base_pitch / 4, dx, dx_pitch / 4, da, db, tokens, stream))
        return cuda_answer(err, "adapter gradient launch");
    return answer(err, QW4_OK, "");
}

static Qwen4Status check_router(const Qwen4MoeConfig *c, const QW4CuTuneWork *w, Qwen4Error *err) {
    if (!c) return answer(err, QW4_INVALID_ARGUMENT, "null config");
    if (!c->experts || !c->top_k || c->top_k > c->experts) return answer(err, QW4_RANGE, "invalid expert count or top_k");
    if (c->experts > w->limits.experts) return answer(err, QW4_CAPACITY, "experts beyond the workspace's");
    return QW4_OK;
}

Qwen4Status qw4cu_balance_forward_device(const Qwen4MoeConfig *c, const float *logits, size_t pitch, const uint32_t *ids, const uint8_t *mask,
                                         size_t tokens, uint32_t *counts, float *prob_sums, float *loss, QW4CuTuneWork *w, Qwen4Error *err) {
    void *stream;
    TRY(usable(w, tokens, &stream, err));
    TRY(check_router(c, w, err));
    Bytes read[3] = {{0}}, out[3];
    const size_t e = c->experts;
    if (tokens) {
        VIEW(logits, tokens, e * 4, pitch, 4, &read[0]);
        VIEW(ids, 1, tokens * c->top_k * 4, tokens * c->top_k * 4, 4, &read[1]);
        if (mask) VIEW(mask, 1, tokens, tokens, 1, &read[2]);
    }
    VIEW(counts, 1, (e + 1) * 4, (e + 1) * 4, 4, &out[0]);
    VIEW(prob_sums, 1, e * 4, e * 4, 4, &out[1]);
    VIEW(loss, 1, 4, 4, 4, &out[2]);
    TRY(apart(out, 3, read, 3, 3, 3, err));
    if (qw4sh_balance_forward(&w->d, c->experts, c->top_k, logits, pitch / 4, ids, mask, tokens, counts, prob_sums, loss, stream))
        return cuda_answer(err, "balance launch");
    return answer(err, QW4_OK, "");
}

Qwen4Status qw4cu_balance_backward_device(const Qwen4MoeConfig *c, const float *logits, size_t pitch, const uint32_t *ids, const uint8_t *mask,
                                          size_t tokens, const uint32_t *counts, float loss_grad, const float *weights_grad, float *grad,
                                          size_t grad_pitch, QW4CuTuneWork *w, Qwen4Error *err) {
    void *stream;
    TRY(usable(w, tokens, &stream, err));
    TRY(check_router(c, w, err));
    if (!tokens) return answer(err, QW4_OK, "");
    Bytes read[5] = {{0}}, out;
    const size_t e = c->experts, pairs = tokens * c->top_k;
    VIEW(logits, tokens, e * 4, pitch, 4, &read[0]);
    VIEW(ids, 1, pairs * 4, pairs * 4, 4, &read[1]);
    if (mask) VIEW(mask, 1, tokens, tokens, 1, &read[2]);
    VIEW(counts, 1, (e + 1) * 4, (e + 1) * 4, 4, &read[3]);
    if (weights_grad) VIEW(weights_grad, 1, pairs * 4, pairs * 4, 4, &read[4]);
    VIEW(grad, tokens, e * 4, grad_pitch, 4, &out);
    TRY(apart(&out, 1, read, 5, 1, 5, err));
    if (qw4sh_balance_backward(&w->d, c->experts, c->top_k, c->norm_topk_prob, logits, pitch / 4, ids, mask, tokens, counts, loss_grad, weights_grad, grad,
                               grad_pitch / 4, stream))
        return cuda_answer(err, "balance gradient launch");
    return answer(err, QW4_OK, "");
}
