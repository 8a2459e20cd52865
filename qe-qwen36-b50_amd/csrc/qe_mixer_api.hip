// C ABI of the token mixers (include/qe_mixer.h): contexts, argument checks, launch plans.
#include <math.h>
#include <string.h>

#include <new>

#include "qe_mixer.h"

#define HIP_TRY(expr)                                                                              \
    do {                                                                                           \
        hipError_t e_ = (expr);                                                                    \
        if (e_ != hipSuccess) return qe_fail(QE_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_));  \
    } while (0)

namespace {

// The context's device for the time of a call, and the caller's again after it.
struct OnDevice {
    int before = -1;
    hipError_t e;
    explicit OnDevice(int device) {
        e = hipGetDevice(&before);
        if (e == hipSuccess && before != device) e = hipSetDevice(device);
        else if (e == hipSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// The word that kernels report into: pinned host memory, so that the host looks without a copy.
struct ErrorWord {
    unsigned *host = nullptr, *dev = nullptr;
    hipError_t make() {
        void *h = nullptr, *d = nullptr;
        hipError_t e = hipHostMalloc(&h, 64, hipHostMallocMapped | hipHostMallocCoherent);
        if (e != hipSuccess) return e;
        host = (unsigned *)h;
        memset(h, 0, 64);
        e = hipHostGetDevicePointer(&d, h, 0);
        dev = (unsigned *)d;
        return e;
    }
    void free() {
        if (host) (void)hipHostFree(host);
        host = nullptr;
    }
    // what was reported since the last look
    int take(const char *where) {
        const unsigned v = __atomic_exchange_n(host, 0u, __ATOMIC_ACQ_REL);
        switch (v) {
            case 0: return QE_OK;
            case QE_BAD_LENGTH:
                return qe_fail(QE_ERR_STATE, "%s: an earlier call met a length or token offset out of range; that sequence's outputs are zeros", where);
            case QE_BAD_PAGE:
                return qe_fail(QE_ERR_STATE, "%s: an earlier call met a page id outside the cache; that sequence's outputs are zeros", where);
            case QE_BAD_SLOT:
                return qe_fail(QE_ERR_STATE, "%s: an earlier call met a slot outside the pool; that sequence's outputs are zeros", where);
            default:
                return qe_fail(QE_ERR_STATE, "%s: in an earlier call a sequence wrote a slot that another one used; the later sequence's outputs are zeros", where);
        }
    }
};

int log2_of(int x) { return __builtin_ctz((unsigned)x); }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
size_t size_of(int type) { return type == QE_F32 ? 4 : 2; }

}  // namespace

struct qe_attn_ctx {
    int device;
    qe_attn_desc d;
    int n_axes;
    float scale_log2;
    ErrorWord err;
    double *turns = nullptr;
    uint8_t *axis = nullptr;
    float *part_o = nullptr;
    float2 *part_ml = nullptr;
    unsigned long long *arrived = nullptr;
};

namespace {

void release(qe_attn_ctx *c) {
    (void)hipFree(c->turns);
    (void)hipFree(c->axis);
    (void)hipFree(c->part_o);
    (void)hipFree(c->part_ml);
    (void)hipFree(c->arrived);
    c->err.free();
    delete c;
}

// Rows of partial results: decode's splits (below QE_ATTN_PART_WGS, each room for the rows of the largest group) or
// prompt's (at most QE_ATTN_WGS tiles of 128 rows).
size_t part_rows() {
    const size_t decode = (size_t)QE_ATTN_PART_WGS * QE_ATTN_GROUP_MAX, prompt = (size_t)QE_ATTN_WGS * 128;
    return decode > prompt ? decode : prompt;
}

int check_batch(const qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, const char *where) {
    if (!c || !b || !kv) return qe_fail(QE_ERR_ARG, "%s: null context, batch or cache", where);
    if (b->n_seqs < 1 || b->n_seqs > 65535) return qe_fail(QE_ERR_ARG, "%s: n_seqs %d is not 1 .. 65535", where, b->n_seqs);
    if (b->n_tokens < 0 || b->n_tokens >= 1 << 24) return qe_fail(QE_ERR_ARG, "%s: n_tokens %d is not 0 .. 2^24 - 1", where, b->n_tokens);
    if (!b->cu_q && b->n_tokens != b->n_seqs)
        return qe_fail(QE_ERR_ARG, "%s: without cu_q n_tokens (%d) is n_seqs (%d)", where, b->n_tokens, b->n_seqs);
    if (!b->kv_len || !b->table) return qe_fail(QE_ERR_ARG, "%s: null kv_len or table", where);
    if (b->max_pages < 1 || (int64_t)b->max_pages * c->d.page > 1 << 30 || b->table_stride < b->max_pages)
        return qe_fail(QE_ERR_ARG, "%s: max_pages %d (of %d positions), table_stride %d", where, b->max_pages, c->d.page, b->table_stride);
    if (b->max_len < 0) return qe_fail(QE_ERR_ARG, "%s: max_len %d", where, b->max_len);
    if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v))
        return qe_fail(QE_ERR_ARG, "%s: cache arrays are null or not 16-byte aligned", where);
    if (kv->n_pages < 1 || kv->n_pages > 0x7fffffff) return qe_fail(QE_ERR_ARG, "%s: n_pages %lld", where, (long long)kv->n_pages);
    return QE_OK;
}

// rows of `width` elements of `type` at p, `stride` apart
int check_rows(const void *p, int64_t stride, int64_t width, int type, const char *what, const char *where) {
    if (!p || !aligned16(p)) return qe_fail(QE_ERR_ARG, "%s: %s is null or not 16-byte aligned", where, what);
    if (stride < width || stride > (int64_t)1 << 32 || stride * (int64_t)size_of(type) % 16)
        return qe_fail(QE_ERR_ARG, "%s: the token stride of %s, %lld, is not a multiple of 16 bytes of at least %lld elements", where, what,
                       (long long)stride, (long long)width);
    return QE_OK;
}

QeAttnArgs attn_args(const qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, const void *q, int64_t q_stride, void *out,
                     int64_t out_stride) {
    QeAttnArgs a{};
    a.q = q; a.out = out; a.kc = kv->k; a.vc = kv->v;
    a.q_stride = q_stride; a.out_stride = out_stride;
    a.cu = b->cu_q; a.kv_len = b->kv_len; a.table = b->table;
    a.n_seqs = b->n_seqs; a.n_tokens = b->n_tokens; a.table_stride = b->table_stride; a.max_pages = b->max_pages;
    a.q_heads = c->d.q_heads; a.kv_heads = c->d.kv_heads; a.group = c->d.q_heads / c->d.kv_heads;
    a.page_log2 = log2_of(c->d.page);
    a.n_pages = (unsigned)kv->n_pages;
    a.scale_log2 = c->scale_log2;
    a.part_o = c->part_o; a.part_ml = c->part_ml; a.arrived = c->arrived;
    a.err = c->err.dev;
    return a;
}

}  // namespace

extern "C" {

int qe_attn_create(int device, const qe_attn_desc *d, qe_attn_ctx **out) {
    if (!d || !out) return qe_fail(QE_ERR_ARG, "qe_attn_create: null argument");
    *out = nullptr;
    if (d->kv_heads < 1 || d->kv_heads > 256 || d->q_heads < 1 || d->q_heads % d->kv_heads || d->q_heads / d->kv_heads > QE_ATTN_GROUP_MAX)
        return qe_fail(QE_ERR_ARG, "qe_attn_create: %d query heads over %d key-value heads", d->q_heads, d->kv_heads);
    if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
        return qe_fail(QE_ERR_ARG, "qe_attn_create: head_dim %d is not 64, 128 or 256", d->head_dim);
    if (d->page < 16 || d->page > 256 || d->page & (d->page - 1))
        return qe_fail(QE_ERR_ARG, "qe_attn_create: page %d is not 16, 32, 64, 128 or 256", d->page);
    if (d->type != QE_F16 && d->type != QE_BF16) return qe_fail(QE_ERR_ARG, "qe_attn_create: type %d", d->type);
    if (!(d->scale >= 0.f) || !isfinite(d->scale)) return qe_fail(QE_ERR_ARG, "qe_attn_create: scale %g", d->scale);
    if (d->rotary < 0 || d->rotary > d->head_dim || d->rotary % 16)
        return qe_fail(QE_ERR_ARG, "qe_attn_create: rotary %d is not a multiple of 16 up to head_dim", d->rotary);
    const int pairs = d->rotary / 2, *s = d->sections;
    if (pairs) {
        if (!(d->theta > 1.0) || !isfinite(d->theta)) return qe_fail(QE_ERR_ARG, "qe_attn_create: theta %g", d->theta);
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0 || s[i] > pairs) return qe_fail(QE_ERR_ARG, "qe_attn_create: sections %d, %d, %d of %d pairs", s[0], s[1], s[2], pairs);
        // taking turns, the height's last pair is 3 (s1 - 1) + 1 and the width's 3 (s2 - 1) + 2
        if (s[0] + s[1] + s[2] != pairs || (d->interleaved && (3 * s[1] - 2 >= pairs || 3 * s[2] - 1 >= pairs)))
            return qe_fail(QE_ERR_ARG, "qe_attn_create: sections %d, %d, %d of %d pairs", s[0], s[1], s[2], pairs);
    }
    OnDevice on(device);
    HIP_TRY(on.e);
    qe_attn_ctx *c = new (std::nothrow) qe_attn_ctx();
    if (!c) return qe_fail(QE_ERR_OOM, "qe_attn_create: out of host memory");
    c->device = device;
    c->d = *d;
    c->n_axes = pairs && (s[1] || s[2]) ? 3 : 1;
    c->scale_log2 = (float)((d->scale ? (double)d->scale : 1.0 / sqrt((double)d->head_dim)) * 1.4426950408889634);
    double turns[128];
    uint8_t axis[128];
    for (int i = 0; i < pairs; ++i) {
        turns[i] = pow(d->theta, -2.0 * i / d->rotary) / 6.283185307179586;
        axis[i] = d->interleaved ? (i % 3 == 1 && i < 3 * s[1] ? 1 : i % 3 == 2 && i < 3 * s[2] ? 2 : 0) : i < s[0] ? 0 : i < s[0] + s[1] ? 1 : 2;
    }
    hipError_t e = c->err.make();
    const size_t rows = part_rows();
    if (e == hipSuccess) e = hipMalloc((void **)&c->turns, sizeof turns);
    if (e == hipSuccess) e = hipMalloc((void **)&c->axis, sizeof axis);
    if (e == hipSuccess) e = hipMalloc((void **)&c->part_o, rows * d->head_dim * 4);
    if (e == hipSuccess) e = hipMalloc((void **)&c->part_ml, rows * sizeof(float2));
    if (e == hipSuccess) e = hipMalloc((void **)&c->arrived, (QE_ATTN_DECODE_WGS + 2) * sizeof(unsigned long long));
    const bool oom = e == hipErrorOutOfMemory;
    if (e == hipSuccess) e = hipMemset(c->arrived, 0, (QE_ATTN_DECODE_WGS + 2) * sizeof(unsigned long long));
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e == hipSuccess && pairs) {
        e = hipMemcpy(c->turns, turns, pairs * sizeof(double), hipMemcpyHostToDevice);
        if (e == hipSuccess) e = hipMemcpy(c->axis, axis, pairs, hipMemcpyHostToDevice);
    }
    if (e != hipSuccess) {
        release(c);
        return qe_fail(oom ? QE_ERR_OOM : QE_ERR_HIP, "qe_attn_create: %s", hipGetErrorString(e));
    }
    *out = c;
    return QE_OK;
}

int qe_attn_destroy(qe_attn_ctx *c) {
    if (!c) return QE_OK;
    OnDevice on(c->device);
    (void)hipDeviceSynchronize();
    release(c);
    return QE_OK;
}

int qe_attn_append(qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, int in_type, const void *q, int64_t q_stride, const void *k,
                   int64_t k_stride, const void *v, int64_t v_stride, const int32_t *pos, void *q_out, int64_t q_out_stride, void *stream) {
    static const char *const where = "qe_attn_append";
    int rc = check_batch(c, b, kv, where);
    if (rc != QE_OK) return rc;
    if (in_type != QE_F32 && in_type != c->d.type) return qe_fail(QE_ERR_ARG, "%s: in_type %d, the cache has type %d", where, in_type, c->d.type);
    if (!q != !q_out) return qe_fail(QE_ERR_ARG, "%s: q and q_out go together", where);
    const int64_t qw = (int64_t)c->d.q_heads * c->d.head_dim, kw = (int64_t)c->d.kv_heads * c->d.head_dim;
    if (b->n_tokens) {
        if (q && (rc = check_rows(q, q_stride, qw, in_type, "q", where)) != QE_OK) return rc;
        if (q && (rc = check_rows(q_out, q_out_stride, qw, c->d.type, "q_out", where)) != QE_OK) return rc;
        if (q == q_out && q && (in_type != c->d.type || q_stride != q_out_stride))
            return qe_fail(QE_ERR_ARG, "%s: q is rotated in place only in the cache's type and with equal strides", where);
        if ((rc = check_rows(k, k_stride, kw, in_type, "k", where)) != QE_OK) return rc;
        if ((rc = check_rows(v, v_stride, kw, in_type, "v", where)) != QE_OK) return rc;
    }
    if ((rc = c->err.take(where)) != QE_OK) return rc;
    if (b->n_tokens == 0) return QE_OK;
    QeAppendArgs a{};
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kc = kv->k; a.vc = kv->v;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
    a.pos = pos; a.cu = b->cu_q; a.kv_len = b->kv_len; a.table = b->table;
    a.turns = c->turns; a.axis = c->axis;
    a.n_axes = c->n_axes; a.n_seqs = b->n_seqs; a.n_tokens = b->n_tokens; a.table_stride = b->table_stride; a.max_pages = b->max_pages;
    a.q_heads = c->d.q_heads; a.kv_heads = c->d.kv_heads; a.head_dim = c->d.head_dim; a.page_log2 = log2_of(c->d.page); a.rotary = c->d.rotary;
    a.n_pages = (unsigned)kv->n_pages;
    a.err = c->err.dev;
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(qe_launch_append(a, in_type, c->d.type, (hipStream_t)stream));
    return QE_OK;
}

static int check_attend(qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, const void *q, int64_t q_stride, const void *out,
                        int64_t out_stride, const char *where) {
    int rc = check_batch(c, b, kv, where);
    if (rc != QE_OK) return rc;
    const int64_t qw = (int64_t)c->d.q_heads * c->d.head_dim;
    if (b->n_tokens) {
        if ((rc = check_rows(q, q_stride, qw, c->d.type, "q", where)) != QE_OK) return rc;
        if ((rc = check_rows(out, out_stride, qw, c->d.type, "out", where)) != QE_OK) return rc;
        if (q == out && q_stride != out_stride) return qe_fail(QE_ERR_ARG, "%s: out is q only with equal strides", where);
    }
    return c->err.take(where);
}

int qe_attn_prompt(qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, const void *q, int64_t q_stride, void *out, int64_t out_stride,
                   void *stream) {
    if (b && !b->cu_q) return qe_fail(QE_ERR_ARG, "qe_attn_prompt: null cu_q (single tokens: qe_attn_decode)");
    const int rc = check_attend(c, b, kv, q, q_stride, out, out_stride, "qe_attn_prompt");
    if (rc != QE_OK || b->n_tokens == 0) return rc;
    QeAttnArgs a = attn_args(c, b, kv, q, q_stride, out, out_stride);
    const int bm = qe_attn_prompt_rows(b->n_tokens, b->n_seqs, a.group, a.kv_heads, c->d.head_dim);
    a.tiles = qe_attn_max_tiles(b->n_tokens, b->n_seqs, a.group, bm);
    if (!qe_fits_launch((int64_t)a.tiles * a.kv_heads, 2 * bm))
        return qe_fail(QE_ERR_ARG, "qe_attn_prompt: %d tokens of %d sequences are more threads than a launch has", b->n_tokens, b->n_seqs);
    const int64_t most = (int64_t)b->max_pages * c->d.page;
    a.splits = qe_attn_prompt_splits((int64_t)a.tiles * a.kv_heads, b->max_len && b->max_len < most ? b->max_len : most);
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(qe_launch_attn_prompt(a, c->d.head_dim, c->d.type, bm, (hipStream_t)stream));
    return QE_OK;
}

int qe_attn_decode(qe_attn_ctx *c, const qe_attn_batch *b, const qe_kv_cache *kv, const void *q, int64_t q_stride, void *out, int64_t out_stride,
                   void *stream) {
    if (b && b->cu_q) return qe_fail(QE_ERR_ARG, "qe_attn_decode: cu_q given (several tokens: qe_attn_prompt)");
    const int rc = check_attend(c, b, kv, q, q_stride, out, out_stride, "qe_attn_decode");
    if (rc != QE_OK) return rc;
    QeAttnArgs a = attn_args(c, b, kv, q, q_stride, out, out_stride);
    const int64_t most = (int64_t)b->max_pages * c->d.page;
    const int64_t max_len = b->max_len && b->max_len < most ? b->max_len : most;
    qe_attn_decode_plan(b->n_seqs, a.kv_heads, c->d.head_dim, max_len, &a.steps, &a.splits);
    a.once = qe_attn_decode_once(b->n_seqs, a.kv_heads, c->d.head_dim, max_len);
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(qe_launch_attn_decode(a, c->d.head_dim, c->d.type, (hipStream_t)stream));
    return QE_OK;
}

int qe_attn_check(qe_attn_ctx *c, void *stream) {
    if (!c) return qe_fail(QE_ERR_ARG, "qe_attn_check: null context");
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
    return c->err.take("qe_attn_check");
}

}  // extern "C"

struct qe_delta_ctx {
    int device;
    qe_delta_desc d;
    float scale;
    ErrorWord err;
    float *ws = nullptr;
    short *ws_kq = nullptr;
    unsigned char *skip = nullptr;
};

static void release(qe_delta_ctx *c) {
    (void)hipFree(c->ws);
    (void)hipFree(c->ws_kq);
    (void)hipFree(c->skip);
    c->err.free();
    delete c;
}

static int delta_args(qe_delta_ctx *c, const qe_delta_args *x, const char *where, QeDeltaArgs *a) {
    if (!c || !x) return qe_fail(QE_ERR_ARG, "%s: null context or arguments", where);
    if (x->n_seqs < 1 || x->n_seqs > c->d.seqs_max) return qe_fail(QE_ERR_ARG, "%s: n_seqs %d is not 1 .. %d", where, x->n_seqs, c->d.seqs_max);
    const int64_t kw = (int64_t)c->d.k_heads * c->d.dim_k, vw = (int64_t)c->d.v_heads * c->d.dim_v;
    int rc;
    if (x->n_tokens) {
        if ((rc = check_rows(x->q, x->q_stride, kw, c->d.type, "q", where)) != QE_OK) return rc;
        if ((rc = check_rows(x->k, x->k_stride, kw, c->d.type, "k", where)) != QE_OK) return rc;
        if ((rc = check_rows(x->v, x->v_stride, vw, c->d.type, "v", where)) != QE_OK) return rc;
        if ((rc = check_rows(x->out, x->out_stride, vw, c->d.type, "out", where)) != QE_OK) return rc;
        if (!x->g || !x->beta) return qe_fail(QE_ERR_ARG, "%s: null g or beta", where);
        if (x->out == x->q || x->out == x->k || x->out == x->v) return qe_fail(QE_ERR_ARG, "%s: out may not be an input", where);
    }
    if (!x->pool || !aligned16(x->pool) || x->n_slots < 1 || x->n_slots > 0x7fffffff)
        return qe_fail(QE_ERR_ARG, "%s: the pool is null, not 16-byte aligned, or of %lld slots", where, (long long)x->n_slots);
    if (!x->slots_in || !x->slots_out) return qe_fail(QE_ERR_ARG, "%s: null slots", where);
    a->q = x->q; a->k = x->k; a->v = x->v; a->out = x->out;
    a->q_stride = x->q_stride; a->k_stride = x->k_stride; a->v_stride = x->v_stride; a->out_stride = x->out_stride;
    a->g = x->g; a->beta = x->beta; a->pool = x->pool; a->n_slots = x->n_slots;
    a->slots_in = x->slots_in; a->slots_out = x->slots_out;
    a->n_seqs = x->n_seqs; a->n_tokens = x->n_tokens;
    a->k_heads = c->d.k_heads; a->v_heads = c->d.v_heads; a->group = c->d.v_heads / c->d.k_heads;
    a->l2norm = c->d.l2norm; a->scale = c->scale;
    a->ws = c->ws; a->ws_kq = c->ws_kq; a->skip = c->skip; a->err = c->err.dev;
    return QE_OK;
}

extern "C" {

int qe_delta_create(int device, const qe_delta_desc *d, qe_delta_ctx **out) {
    if (!d || !out) return qe_fail(QE_ERR_ARG, "qe_delta_create: null argument");
    *out = nullptr;
    if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads > 1024 || d->v_heads % d->k_heads)
        return qe_fail(QE_ERR_ARG, "qe_delta_create: %d value heads over %d key heads", d->v_heads, d->k_heads);
    if ((d->dim_k != 64 && d->dim_k != 128) || (d->dim_v != 64 && d->dim_v != 128))
        return qe_fail(QE_ERR_ARG, "qe_delta_create: dimensions %d and %d are not 64 or 128", d->dim_k, d->dim_v);
    if (d->type != QE_F32 && d->type != QE_F16 && d->type != QE_BF16) return qe_fail(QE_ERR_ARG, "qe_delta_create: type %d", d->type);
    if (!(d->scale >= 0.f) || !isfinite(d->scale)) return qe_fail(QE_ERR_ARG, "qe_delta_create: scale %g", d->scale);
    if (d->t_max < 1 || d->t_max > 1 << 20 || d->seqs_max < 1 || d->seqs_max > 65535)
        return qe_fail(QE_ERR_ARG, "qe_delta_create: t_max %d, seqs_max %d", d->t_max, d->seqs_max);
    OnDevice on(device);
    HIP_TRY(on.e);
    qe_delta_ctx *c = new (std::nothrow) qe_delta_ctx();
    if (!c) return qe_fail(QE_ERR_OOM, "qe_delta_create: out of host memory");
    c->device = device;
    c->d = *d;
    c->scale = d->scale ? d->scale : (float)(1.0 / sqrt((double)d->dim_k));
    hipError_t e = c->err.make();
    const size_t chunks = (size_t)qe_delta_max_chunks(d->t_max, d->seqs_max);
    if (e == hipSuccess) e = hipMalloc((void **)&c->ws, chunks * d->v_heads * QE_DELTA_WS * 4);
    const size_t kept = (size_t)qe_delta_kept_planes((int)size_of(d->type), d->type == QE_BF16) * 2 * QE_DELTA_C * d->dim_k * 2;
    if (e == hipSuccess && kept) e = hipMalloc((void **)&c->ws_kq, chunks * d->k_heads * kept);
    if (e == hipSuccess) e = hipMalloc((void **)&c->skip, (size_t)d->seqs_max);
    if (e != hipSuccess) {
        release(c);
        return qe_fail(e == hipErrorOutOfMemory ? QE_ERR_OOM : QE_ERR_HIP, "qe_delta_create: %s", hipGetErrorString(e));
    }
    *out = c;
    return QE_OK;
}

int qe_delta_destroy(qe_delta_ctx *c) {
    if (!c) return QE_OK;
    OnDevice on(c->device);
    (void)hipDeviceSynchronize();
    release(c);
    return QE_OK;
}

int qe_delta_prompt(qe_delta_ctx *c, const qe_delta_args *x, const int32_t *cu, void *stream) {
    static const char *const where = "qe_delta_prompt";
    QeDeltaArgs a{};
    int rc = delta_args(c, x, where, &a);
    if (rc != QE_OK) return rc;
    if (!cu) return qe_fail(QE_ERR_ARG, "%s: null cu (single tokens: qe_delta_decode)", where);
    if (x->n_tokens < 0 || x->n_tokens > c->d.t_max) return qe_fail(QE_ERR_ARG, "%s: n_tokens %d is not 0 .. %d", where, x->n_tokens, c->d.t_max);
    const int64_t chunks = qe_delta_max_chunks(x->n_tokens, x->n_seqs);
    if (!qe_fits_launch((int64_t)x->n_seqs * c->d.v_heads * (c->d.dim_v / 16), 512) || !qe_fits_launch(chunks * c->d.v_heads, 256))
        return qe_fail(QE_ERR_ARG, "%s: %d tokens of %d sequences are more threads than a launch has", where, x->n_tokens, x->n_seqs);
    if ((rc = c->err.take(where)) != QE_OK) return rc;
    a.cu = cu;
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(qe_launch_delta_prompt(a, c->d.dim_k, c->d.dim_v, c->d.type, (hipStream_t)stream));
    return QE_OK;
}

int qe_delta_decode(qe_delta_ctx *c, const qe_delta_args *x, void *stream) {
    static const char *const where = "qe_delta_decode";
    QeDeltaArgs a{};
    int rc = delta_args(c, x, where, &a);
    if (rc != QE_OK) return rc;
    if (x->n_tokens != x->n_seqs) return qe_fail(QE_ERR_ARG, "%s: n_tokens %d, n_seqs %d", where, x->n_tokens, x->n_seqs);
    if (!qe_fits_launch((int64_t)x->n_seqs * c->d.v_heads * (c->d.dim_v / 32), 256))
        return qe_fail(QE_ERR_ARG, "%s: %d sequences are more threads than a launch has", where, x->n_seqs);
    if ((rc = c->err.take(where)) != QE_OK) return rc;
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(qe_launch_delta_decode(a, c->d.dim_k, c->d.dim_v, c->d.type, (hipStream_t)stream));
    return QE_OK;
}

int qe_delta_check(qe_delta_ctx *c, void *stream) {
    if (!c) return qe_fail(QE_ERR_ARG, "qe_delta_check: null context");
    OnDevice on(c->device);
    HIP_TRY(on.e);
    HIP_TRY(hipStreamSynchronize((hipStream_t)stream));
    return c->err.take("qe_delta_check");
}

}  // extern "C"
