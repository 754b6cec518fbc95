// C ABI of the attention on token sequences: argument checks and dispatch.
#include "seq_umma.cuh"

namespace ca {

int check_seq_dtype(int dtype) {
    if (dtype == CA_F32 || dtype == CA_BF16 || dtype == CA_F16) return CA_OK;
    set_error("dtype %d: Float32, BFloat16 and Float16 are supported", dtype);
    return CA_ERR_BAD_DESC;
}

static int check_strided(const void* p, const int64_t* strides, int dtype, const char* name, bool used) {
    const int64_t e = dtype == CA_F32 ? 4 : 2;
    if (used && !p) { set_error("%s has no data (NULL)", name); return CA_ERR_NULL; }
    if (reinterpret_cast<uintptr_t>(p) % 16) { set_error("%s is not 16-byte aligned", name); return CA_ERR_BAD_DESC; }
    for (int i = 0; i < 3; ++i)
        if (strides[i] < 0 || strides[i] * e % 16 || strides[i] > (1LL << 40) / e - 1) {
            set_error("%s: stride of %lld elements (multiples of 16 bytes below 2^40 are supported)", name, (long long)strides[i]);
            return CA_ERR_BAD_DESC;
        }
    return CA_OK;
}

int check_view(const ca_seq_view* v, int dtype, const char* name, bool used) {
    if (!v) { set_error("%s is NULL", name); return CA_ERR_NULL; }
    const int64_t s[3] = {v->head, v->token, v->batch};
    return check_strided(v->data, s, dtype, name, used);
}

int check_page_view(const ca_page_view* v, int dtype, const char* name, bool used) {
    if (!v) { set_error("%s is NULL", name); return CA_ERR_NULL; }
    const int64_t s[3] = {v->token, v->head, v->page};
    return check_strided(v->data, s, dtype, name, used);
}

int check_pages(const ca_pages* p, int tokens) {
    if (!p) { set_error("pages is NULL"); return CA_ERR_NULL; }
    if (p->sequences < 0 || p->width < 0 || p->pages < 0) { set_error("sequences=%d width=%d pages=%d must not be negative", p->sequences, p->width, p->pages); return CA_ERR_BAD_DESC; }
    if (p->page < 16 || p->page % 16) { set_error("page=%d: multiples of 16 tokens are supported", p->page); return CA_ERR_BAD_DESC; }
    if (tokens && !p->sequences) { set_error("%d tokens of no sequence", tokens); return CA_ERR_BAD_DESC; }
    if (tokens && (!p->table || !p->starts || !p->lengths)) { set_error("table, starts and lengths must not be NULL"); return CA_ERR_NULL; }
    return CA_OK;
}

static int fill(const ca_seq_desc* d, SeqArgs* a) {
    if (!d) { set_error("descriptor is NULL"); return CA_ERR_NULL; }
    const int rc = check_seq_dtype(d->dtype);
    if (rc) return rc;
    if (d->dim < 8 || d->dim % 8 || d->dim > 128) { set_error("dim=%d: multiples of 8 up to 128 are supported", d->dim); return CA_ERR_BAD_DESC; }
    if (d->heads_q < 1 || d->heads_kv < 1 || d->heads_q % d->heads_kv) {
        set_error("heads_q=%d must be a positive multiple of heads_kv=%d", d->heads_q, d->heads_kv);
        return CA_ERR_BAD_DESC;
    }
    if (d->tokens < 0 || d->batch < 0) { set_error("tokens=%d batch=%d must not be negative", d->tokens, d->batch); return CA_ERR_BAD_DESC; }
    if (d->right < 0 || d->sinks < 0) { set_error("right=%d sinks=%d must not be negative", d->right, d->sinks); return CA_ERR_BAD_DESC; }
    a->G = d->heads_q / d->heads_kv;
    if (d->tokens > kNoLeft || (int64_t)d->tokens * a->G > INT32_MAX - 256 || d->heads_kv > 65535 || d->batch > 65535) {
        set_error("tokens=%d heads=%d/%d batch=%d exceed 2^31 rows per key head or the grid limit 65535", d->tokens, d->heads_q, d->heads_kv, d->batch);
        return CA_ERR_TOO_LARGE;
    }
    // ceil(2^(31 + s) / G) with 2^s >= G: off by less than 2^s / 2^(31 + s) = 2^-31 of a unit per row, so the quotient is exact
    int shift = 0;
    while ((1LL << shift) < a->G) ++shift;
    a->g_shift = 31 + shift;
    a->g_mul = (uint32_t)(((1ULL << (31 + shift)) + a->G - 1) / a->G);
    a->D = d->dim; a->Hq = d->heads_q; a->Hkv = d->heads_kv;
    a->N = d->tokens; a->B = d->batch;
    a->left = d->left < 0 || d->left > kNoLeft ? kNoLeft : d->left;
    a->right = d->right > kNoLeft ? kNoLeft : d->right;
    a->sinks = d->sinks;
    a->scale = d->scale;
    if (!isfinite(d->scale)) { set_error("scale is not finite"); return CA_ERR_BAD_DESC; }
    a->scale_log2 = d->scale * kLog2e;
    a->mag_log2 = fmaxf(fabsf(a->scale_log2), 1e-30f);
    a->status = status_word();
    return CA_OK;
}

// delta, one float a row, padded so that what follows is aligned
static size_t delta_bytes(const SeqArgs& a) { return ((size_t)a.N * a.B * a.Hq * sizeof(float) + 255) & ~(size_t)255; }

}  // namespace ca

using namespace ca;

extern "C" {

int ca_window_fwd(const ca_seq_desc* d, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                  const int32_t* lengths, const ca_seq_view* y, const ca_seq_view* y_rest, float* lse, void* stream) {
    SeqArgs a{};
    int rc = fill(d, &a);
    if (rc) return rc;
    const bool some = a.N && a.B;
    if ((rc = check_view(q, d->dtype, "q", some)) || (rc = check_view(k, d->dtype, "k", some)) || (rc = check_view(v, d->dtype, "v", some)) ||
        (rc = check_view(y, d->dtype, "y", some)) || (y_rest && (rc = check_view(y_rest, d->dtype, "y_rest", false))))
        return rc;
    if (!some) return CA_OK;
    a.q = *q; a.k = *k; a.v = *v; a.y = *y;
    if (y_rest) a.rest = *y_rest;
    a.lengths = lengths;
    a.lse = lse;
    return d->dtype == CA_F32 ? fma_fwd(a, as_stream(stream)) : umma_window_fwd(a, d->dtype, as_stream(stream));
}

size_t ca_window_bwd_workspace(const ca_seq_desc* d) {
    SeqArgs a{};
    if (fill(d, &a)) return 0;
    return delta_bytes(a) + (d->dtype == CA_F32 ? fma_bwd_parts(a) : umma_bwd_parts(a));
}

int ca_window_bwd(const ca_seq_desc* d, const ca_seq_view* q, const ca_seq_view* k, const ca_seq_view* v,
                  const ca_seq_view* y, const ca_seq_view* y_rest, const ca_seq_view* dy, const int32_t* lengths, const float* lse,
                  const ca_seq_view* dq, const ca_seq_view* dk, const ca_seq_view* dv, void* workspace, void* stream) {
    SeqArgs a{};
    int rc = fill(d, &a);
    if (rc) return rc;
    const bool some = a.N && a.B;
    if ((rc = check_view(q, d->dtype, "q", some)) || (rc = check_view(k, d->dtype, "k", some)) || (rc = check_view(v, d->dtype, "v", some)) ||
        (rc = check_view(y, d->dtype, "y", some)) || (rc = check_view(dy, d->dtype, "dy", some)) || (rc = check_view(dq, d->dtype, "dq", some)) ||
        (rc = check_view(dk, d->dtype, "dk", some)) || (rc = check_view(dv, d->dtype, "dv", some)) || (y_rest && (rc = check_view(y_rest, d->dtype, "y_rest", false))))
        return rc;
    if (!some) return CA_OK;
    if (!lse || !workspace) { set_error("lse and workspace must not be NULL"); return CA_ERR_NULL; }
    if (reinterpret_cast<uintptr_t>(workspace) % 16) { set_error("workspace is not 16-byte aligned"); return CA_ERR_BAD_DESC; }
    a.q = *q; a.k = *k; a.v = *v; a.y = *y; a.dy = *dy; a.dq = *dq; a.dk = *dk; a.dv = *dv;
    if (y_rest) a.rest = *y_rest;
    a.lengths = lengths;
    a.lse = const_cast<float*>(lse);
    a.delta = static_cast<float*>(workspace);
    float* parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + delta_bytes(a));
    return d->dtype == CA_F32 ? fma_bwd(a, parts, as_stream(stream)) : umma_window_bwd(a, d->dtype, parts, as_stream(stream));
}

int ca_paged_window(const ca_seq_desc* d, const ca_seq_view* q, const ca_page_view* k_pages, const ca_page_view* v_pages,
                    const ca_pages* pages, const ca_seq_view* y, void* stream) {
    SeqArgs a{};
    int rc = fill(d, &a);
    if (rc) return rc;
    const bool some = a.N && a.B;
    if (d->batch != 1) { set_error("packed tokens have batch 1 (got %d)", d->batch); return CA_ERR_BAD_DESC; }
    if (d->right) { set_error("right=%d: a cache holds no later tokens", d->right); return CA_ERR_BAD_DESC; }
    if ((rc = check_pages(pages, d->tokens)) || (rc = check_view(q, d->dtype, "q", some)) || (rc = check_view(y, d->dtype, "y", some)) ||
        (rc = check_page_view(k_pages, d->dtype, "k_pages", some && pages->pages)) || (rc = check_page_view(v_pages, d->dtype, "v_pages", some && pages->pages)))
        return rc;
    if (!some) return CA_OK;
    a.q = *q; a.y = *y;
    a.kp = *k_pages; a.vp = *v_pages;
    a.pages = *pages;
    // Few rows a key head, on average: the keys are what counts.  More than one tile of 16 rows reads them again, from L2; beyond
    // four the tiles of 128 (64) rows win.  That is so for sequences alike: a mixed call goes one way as a whole and pays for it (63
    // single tokens 98 us, a chunk of 900 93 us, both in one call 385; with a chunk of 1000, by the other kernel, 275).
    if ((int64_t)a.N * a.G <= 64LL * a.pages.sequences || !a.pages.pages) return decode_paged(a, d->dtype, as_stream(stream));
    return d->dtype == CA_F32 ? fma_fwd(a, as_stream(stream)) : umma_paged(a, d->dtype, as_stream(stream));
}

}  // extern "C"
