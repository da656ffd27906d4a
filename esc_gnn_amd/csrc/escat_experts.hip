// escat_experts.hip -- entry points of the experts' products (include/escat.h): argument checks and workspaces
#include "escat_experts.h"

__attribute__((visibility("hidden"))) int escat_experts_rows_fwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1,
                           const void *w2, const void *b2, void *h, float *u, float *part, void *y, hipStream_t st);
__attribute__((visibility("hidden"))) int escat_experts_rows_bwd(int type, const EDims &n, const EPlan &p, const void *x, const float *weights, const void *w1, const void *b1,
                           const void *w2, const void *b2, const void *dy, void *h, void *du, float *u, float *part, float *dwp, float *ws, void *dx, float *dw, hipStream_t st);
__attribute__((visibility("hidden"))) int escat_experts_grad_chunk(int type, int64_t P, int E, int M, int N);
__attribute__((visibility("hidden"))) int64_t escat_experts_grad_chunks(int64_t P, int E, int chunk);
__attribute__((visibility("hidden"))) int escat_experts_plan_by_expert(const EPlan &p, int64_t rows, int E, const EPlan &by, hipStream_t st);
__attribute__((visibility("hidden"))) int escat_experts_grad(int type, const EDims &n, const EPlan &p, const int *at, bool w2, const void *a, const void *b, const float *weights, int M, int N,
                       int chunk, float *part, void *out, void *db, hipStream_t st);

__attribute__((visibility("hidden"))) bool escat_experts_few(int type, const EDims &n);
__attribute__((visibility("hidden"))) int escat_experts_few_fwd(int type, const EDims &n, const int *experts, const void *x, const float *weights, const void *w1, const void *b1,
                          const void *w2, const void *b2, float *h, void *y, hipStream_t st);

static int check_dims(const char *who, const escat_experts_dims *n)
{
    if (!n) return fail(ESCAT_EINVAL, "%s: dims is null", who);
    if (!escat_type_bytes(n->type)) return fail(ESCAT_EINVAL, "%s: type = %d", who, n->type);
    if (n->rows < 0 || n->d < 1 || n->h < 1 || n->o < 1 || n->experts < 1 || n->k < 1)
        return fail(ESCAT_EINVAL, "%s: rows = %lld, d = %d, h = %d, o = %d, experts = %d, k = %d", who, (long long)n->rows, n->d, n->h, n->o, n->experts, n->k);
    const int least = 16 / escat_type_bytes(n->type);
    if (n->d < least || n->h < least || n->o < least) return fail(ESCAT_ERANGE, "%s: d = %d, h = %d, o = %d: rows of at least 16 bytes (%d elements)", who, n->d, n->h, n->o, least);
    if ((int64_t)n->h * (n->d > n->o ? n->d : n->o) > 0x3fffffff || (int64_t)n->h * n->k > 0x7fffff)
        return fail(ESCAT_ERANGE, "%s: h = %d by d = %d and o = %d (below 2^30 elements a matrix), k = %d (h k below 2^23)", who, n->h, n->d, n->o, n->k);
    if (n->experts > ESCAT_ROUTE_MAX_EXPERTS || n->k > 64 || n->rows > 0x3fffffff / n->k || n->d > 65536 || n->h > 65536 || n->o > 65536)
        return fail(ESCAT_ERANGE, "%s: rows * k = %lld * %d (below 2^30), experts = %d (at most %d), k at most 64, d = %d, h = %d, o = %d (at most 65536)", who,
                    (long long)n->rows, n->k, n->experts, ESCAT_ROUTE_MAX_EXPERTS, n->d, n->h, n->o);
    return ESCAT_OK;
}
static EDims dims_of(const escat_experts_dims *n) { return {n->rows, n->d, n->h, n->o, n->experts, n->k}; }
static size_t up(size_t b) { return (b + 255) & ~(size_t)255; }

// workspace of the forward: h (unless the caller keeps it) | by pair: results of the pairs;  of the backward: h (unless kept) | du | by pair: results of the pairs, by combination:
// positions sorted by expert | parts of dw | weights by position | chunks of the
// weight gradients (one after the other in the same place)
static size_t part_bytes(const escat_experts_dims *n, int M) { return combo_keys(n->rows, n->experts, n->k) ? 0 : up((size_t)n->rows * n->k * M * 4); }
// a second plan, by pair, of a plan by combination (k = 1: the first serves)
static size_t by_expert_bytes(const escat_experts_dims *n)
{
    if (!combo_keys(n->rows, n->experts, n->k) || n->k == 1) return 0;
    int64_t ints;
    plan_view(nullptr, n->rows * n->k, 1, n->experts, 0, &ints);
    return up((size_t)(ints + (int64_t)combo_keys(n->rows, n->experts, n->k) * n->k) * 4);             // and where each key's runs begin
}
static size_t hidden_bytes(const escat_experts_dims *n) { return up((size_t)n->rows * n->k * n->h * escat_type_bytes(n->type)); }
static size_t chunk_bytes(const escat_experts_dims *n, int M, int N)
{
    const int64_t P = n->rows * n->k;
    const int c = escat_experts_grad_chunk(n->type, P, n->experts, M, N);
    return c ? up((size_t)escat_experts_grad_chunks(P, n->experts, c) * ((size_t)M * N + N) * 4) : 0;
}

extern "C" size_t escat_experts_hidden_bytes(const escat_experts_dims *n) { return check_dims("escat_experts_hidden_bytes", n) ? 0 : hidden_bytes(n) + (keeps_u(n->type, n->d) ? up((size_t)n->rows * n->k * n->h * 4) : 0) + 256; }

extern "C" size_t escat_experts_workspace_bytes(const escat_experts_dims *n, int backward, int hidden)
{
    if (check_dims("escat_experts_workspace_bytes", n)) return 0;
    const size_t own = hidden ? 0 : hidden_bytes(n);
    if (!backward && escat_experts_few(n->type, dims_of(n))) return up((size_t)n->rows * n->k * n->h * 4) + 256;
    if (!backward) return own + part_bytes(n, n->o) + 256;
    const size_t c1 = chunk_bytes(n, n->d, n->h), c2 = chunk_bytes(n, n->h, n->o);
    return own + hidden_bytes(n) + part_bytes(n, n->d) + by_expert_bytes(n) + up((size_t)((n->h + XN - 1) / XN) * n->rows * n->k * 4) + up((size_t)n->rows * n->k * 4) + (c1 > c2 ? c1 : c2) + 256;
}

extern "C" int escat_experts_fwd_needs_plan(const escat_experts_dims *n)
{
    if (check_dims("escat_experts_fwd_needs_plan", n)) return 1;
    return escat_experts_few(n->type, dims_of(n)) ? 0 : 1;
}

extern "C" int escat_experts_fwd(const escat_experts_dims *n, const void *x, const float *weights, const int32_t *experts_of_rows, const void *w1, const void *b1,
                                 const void *w2, const void *b2, const void *plan, void *y, void *hidden, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_dims("escat_experts_fwd", n); if (rc) return rc;
    if (n->rows == 0) return ESCAT_OK;
    const bool few = escat_experts_few(n->type, dims_of(n));
    if (!x || !weights || !w1 || !w2 || !y || (few ? !experts_of_rows : !plan)) return fail(ESCAT_EINVAL, "escat_experts_fwd: null pointer");
    if (hidden && ((uintptr_t)hidden & 15)) return fail(ESCAT_EINVAL, "escat_experts: hidden is not aligned to 16 bytes");
    if (!workspace || workspace_bytes < escat_experts_workspace_bytes(n, 0, hidden != nullptr) || ((uintptr_t)workspace & 15))
        return fail(ESCAT_EWORKSPACE, "escat_experts_fwd: workspace of %zu bytes (16-byte aligned), needs %zu", workspace_bytes, escat_experts_workspace_bytes(n, 0, hidden != nullptr));
    char *ws = (char *)workspace;
    if (few) return escat_experts_few_fwd(n->type, dims_of(n), experts_of_rows, x, weights, w1, b1, w2, b2, (float *)ws, y, (hipStream_t)stream);
    const EPlan p = plan_of(const_cast<void *>(plan), n->rows, n->k, n->experts);
    void *h = hidden;
    if (!h) { h = ws; ws += hidden_bytes(n); }
    return escat_experts_rows_fwd(n->type, dims_of(n), p, x, weights, w1, b1, w2, b2, h, hidden && keeps_u(n->type, n->d) ? (float *)((char *)hidden + hidden_bytes(n)) : nullptr, (float *)ws, y, (hipStream_t)stream);
}

extern "C" int escat_experts_bwd(const escat_experts_dims *n, const void *x, const float *weights, const void *w1, const void *b1, const void *w2,
                                 const void *b2, const void *plan, const void *hidden, const void *dy, void *dx, float *dweights, void *dw1, void *db1, void *dw2, void *db2,
                                 void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_dims("escat_experts_bwd", n); if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (!w1 || !w2 || !plan) return fail(ESCAT_EINVAL, "escat_experts_bwd: null pointer");
    if (n->rows > 0 && (!x || !weights || !dy)) return fail(ESCAT_EINVAL, "escat_experts_bwd: null pointer");
    if ((db1 && !dw1) || (db2 && !dw2)) return fail(ESCAT_EINVAL, "escat_experts_bwd: a bias's gradient comes with its weight's");
    if (hidden && ((uintptr_t)hidden & 15)) return fail(ESCAT_EINVAL, "escat_experts: hidden is not aligned to 16 bytes");
    if (!workspace || workspace_bytes < escat_experts_workspace_bytes(n, 1, hidden != nullptr) || ((uintptr_t)workspace & 15))
        return fail(ESCAT_EWORKSPACE, "escat_experts_bwd: workspace of %zu bytes (16-byte aligned), needs %zu", workspace_bytes, escat_experts_workspace_bytes(n, 1, hidden != nullptr));
    const int64_t P = n->rows * n->k;
    char *ws = (char *)workspace;
    void *h = const_cast<void *>(hidden);
    if (!h) { h = ws; ws += hidden_bytes(n); }
    void *du = ws; ws += hidden_bytes(n);
    float *part = (float *)ws; ws += part_bytes(n, n->d);
    void *by_mem = ws; ws += by_expert_bytes(n);
    float *dwp = (float *)ws; ws += up((size_t)((n->h + XN - 1) / XN) * P * 4);
    float *sw = (float *)ws; ws += up((size_t)P * 4);
    float *chunks = (float *)ws;
    const EDims d = dims_of(n);
    const EPlan p = plan_of(const_cast<void *>(plan), n->rows, n->k, n->experts);
    if (n->rows > 0) { rc = escat_experts_rows_bwd(n->type, d, p, x, weights, w1, b1, w2, b2, dy, hidden || !dw2 ? nullptr : h, du,
                                                      hidden && keeps_u(n->type, n->d) ? (float *)((char *)const_cast<void *>(hidden) + hidden_bytes(n)) : nullptr, part, dwp, sw, dx, dweights, st); if (rc) return rc; }
    // the weights' gradients (without rows: zeros) sum by expert
    EPlan by = p;
    const int *at = nullptr;
    if (p.base && n->k > 1 && (dw1 || dw2)) {
        int64_t ints;
        by = plan_view(by_mem, P, 1, n->experts, 0, &ints);
        by.hist = (int *)by_mem + ints;
        rc = escat_experts_plan_by_expert(p, n->rows, n->experts, by, st); if (rc) return rc;
        at = by.pair;
    }
    if (dw2) { rc = escat_experts_grad(n->type, d, by, at, true, h, dy, sw, n->h, n->o, escat_experts_grad_chunk(n->type, P, n->experts, n->h, n->o), chunks, dw2, db2, st); if (rc) return rc; }
    if (dw1) { rc = escat_experts_grad(n->type, d, by, at, false, x, du, sw, n->d, n->h, escat_experts_grad_chunk(n->type, P, n->experts, n->d, n->h), chunks, dw1, db1, st); if (rc) return rc; }
    return ESCAT_OK;
}
