// Rotary positions with several axes, and their serving form that also stores k and v into a paged cache.
//
// Pair p of a head is the complex number a + ib, multiplied by exp(2 pi i f_p x), x the integer position on the pair's
// axis.  f_p is kept as F_p = f_p 2^64 modulo 2^64: F_p x modulo 2^64 is the exact phase modulo one turn for every
// 32-bit position, one wrapping multiplication, where a Float32 product would be off by 2^-24 of the whole angle (0.006
// at position 10^5).  Its upper 32 bits, a signed fraction of half a turn, go to sincospi.  The gradient is the rotation
// back, so the backward is the same kernel.
//
// Bound: bytes.  A token's sines and cosines are shared by all of its heads, so a block computes them once for a few
// tokens, keeps them in shared memory and then streams the heads of all tensors through 16-byte loads and stores.  Measured:
// 2 x 16384 tokens, 20 heads of 128 features, bfloat16: 60 us, 5.6 TB/s (issue slots 73 % taken); two heads at a time for more
// bytes under way took 93 us for what takes 68.
#include "seq.cuh"

namespace ca {
namespace {

struct RotaryTensor {
    const void* src;
    void* dst;
    int64_t s_head, s_token, s_batch;
    int64_t d_head, d_token, d_batch;     // into a cache: d_batch is the stride of a page
    int heads, turn, paged;
};

struct RotaryArgs {
    RotaryTensor t[3];
    int nt, total_heads;
    uint32_t heads_inv;                   // ceil(2^32 / total_heads): exact quotients of items below 2^32 / total_heads
    int D, R, axes, ends[CA_MAX_AXES];    // ends: first pair behind each section
    const int* pos;
    int64_t p_axis, p_token, p_batch;
    const int64_t* turns;
    int N;
    int64_t tokens;                       // N * B
    float sign;
    int per_block;                        // tokens of a block
    ca_pages pages;
};

constexpr int kRotaryThreads = 256, kRotaryTokens = 8;

// V elements of T at a time (16 bytes where the pairs and the rest divide so, else less).
template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T e[V]; };

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRotaryThreads, 8) rotary_kernel(const __grid_constant__ RotaryArgs a) {
    extern __shared__ float2 cs[];                    // [token][p % V][p / V]: lanes of consecutive chunks read consecutive words
    __shared__ int s_page[kRotaryTokens], s_off[kRotaryTokens], s_batch[kRotaryTokens], s_token[kRotaryTokens];
    const int R = a.R, nc = R / V;
    const int64_t tok0 = (int64_t)blockIdx.x * a.per_block;
    const int ntok = (int)min((int64_t)a.per_block, a.tokens - tok0);
    // Quotients are taken once a token: as part of every piece they were more than half of the instructions.
    if (threadIdx.x < ntok) {
        const uint32_t tok = (uint32_t)tok0 + threadIdx.x, b = tok / (uint32_t)a.N;
        s_batch[threadIdx.x] = (int)b;
        s_token[threadIdx.x] = (int)(tok - b * (uint32_t)a.N);
    }
    __syncthreads();

    for (int i = threadIdx.x; i < ntok * R; i += kRotaryThreads) {
        const int t = i / R, p = i - t * R;
        const int64_t b = s_batch[t], n = s_token[t];
        int axis = 0;
        while (axis + 1 < a.axes && p >= a.ends[axis]) ++axis;
        const int x = a.pos[axis * a.p_axis + n * a.p_token + b * a.p_batch];
        const uint64_t phase = (uint64_t)(int64_t)x * (uint64_t)a.turns[p];
        float s, c;
        sincospif((float)(int32_t)(phase >> 32) * 4.656612873077393e-10f, &s, &c);       // 2^-31: in half turns
        cs[(size_t)t * R + (p % V) * nc + p / V] = make_float2(c, a.sign * s);
    }
    if (a.pages.table && threadIdx.x < ntok) {        // where the token lives in the cache
        const int tok = (int)tok0 + threadIdx.x;
        int lo = 0, hi = a.pages.sequences;           // the last sequence whose start is <= tok
        while (lo + 1 < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.pages.starts[mid] <= tok) lo = mid; else hi = mid;
        }
        const int64_t j = (int64_t)a.pages.lengths[lo] - a.pages.starts[lo + 1] + tok;
        int page = -1, off = 0;
        if (tok >= a.pages.starts[lo] && tok < a.pages.starts[lo + 1] && j >= 0 && j / a.pages.page < a.pages.width) {
            page = a.pages.table[j / a.pages.page + (int64_t)a.pages.width * lo];
            off = (int)(j % a.pages.page);
            if (page >= a.pages.pages) page = -1;
        }
        s_page[threadIdx.x] = page;
        s_off[threadIdx.x] = off;
    }
    __syncthreads();

    // A group of nv threads takes one head of one token: R/V chunks of pairs, then the features that pass.
    const int nv = nc + (a.D - 2 * R) / V;
    const int groups = max(1, kRotaryThreads / nv);
    const int g0 = (int)threadIdx.x / nv;
    if (g0 >= groups) return;
    for (int c = threadIdx.x - g0 * nv; c < nv; c += groups == 1 ? kRotaryThreads : nv) {
        for (int item = g0; item < ntok * a.total_heads; item += groups) {
            const int t = a.total_heads == 1 ? item : (int)__umulhi((uint32_t)item, a.heads_inv);
            int h = item - t * a.total_heads, which = 0;
            while (which + 1 < a.nt && h >= a.t[which].heads) h -= a.t[which++].heads;
            const RotaryTensor& x = a.t[which];
            const int64_t b = s_batch[t], n = s_token[t];
            const T* src = (const T*)x.src + h * x.s_head + n * x.s_token + b * x.s_batch;
            T* dst;
            if (x.paged) {
                if (s_page[t] < 0) continue;
                dst = (T*)x.dst + h * x.d_head + s_off[t] * x.d_token + s_page[t] * x.d_batch;
            } else {
                dst = (T*)x.dst + h * x.d_head + n * x.d_token + b * x.d_batch;
            }
            typedef Vec<T, V> W;
            if (c >= nc) {
                const int f = 2 * R + (c - nc) * V;
                *(W*)(dst + f) = *(const W*)(src + f);
                continue;
            }
            const int fa = INTER ? 2 * c * V : c * V, fb = INTER ? fa + V : R + fa;
            const W u = *(const W*)(src + fa), w = *(const W*)(src + fb);
            W ou = u, ow = w;
            if (x.turn) {
                const float2* q = cs + (size_t)t * R + c;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float2 e = q[i * nc];
                    const float re = INTER ? to_float(2 * i < V ? u.e[(2 * i) % V] : w.e[(2 * i) % V]) : to_float(u.e[i]);
                    const float im = INTER ? to_float(2 * i < V ? (V > 1 ? u.e[(2 * i + 1) % V] : w.e[0]) : w.e[(2 * i + 1) % V])
                                           : to_float(w.e[i]);
                    const float nr = re * e.x - im * e.y, ni = re * e.y + im * e.x;
                    if (!INTER) {
                        ou.e[i] = from_float<T>(nr);
                        ow.e[i] = from_float<T>(ni);
                    } else if (V == 1) {
                        ou.e[0] = from_float<T>(nr);
                        ow.e[0] = from_float<T>(ni);
                    } else if (2 * i < V) {
                        ou.e[(2 * i) % V] = from_float<T>(nr);
                        ou.e[(2 * i + 1) % V] = from_float<T>(ni);
                    } else {
                        ow.e[(2 * i) % V] = from_float<T>(nr);
                        ow.e[(2 * i + 1) % V] = from_float<T>(ni);
                    }
                }
            }
            *(W*)(dst + fa) = ou;
            *(W*)(dst + fb) = ow;
        }
    }
}

template <typename T, int V>
int launch_rotary(const RotaryArgs& a, bool interleaved, cudaStream_t st) {
    const size_t smem = (size_t)a.per_block * a.R * sizeof(float2);
    const unsigned blocks = (unsigned)((a.tokens + a.per_block - 1) / a.per_block);
    if (interleaved) rotary_kernel<T, V, true><<<blocks, kRotaryThreads, smem, st>>>(a);
    else rotary_kernel<T, V, false><<<blocks, kRotaryThreads, smem, st>>>(a);
    CA_CHECK_LAUNCH("rotary kernel");
    return CA_OK;
}

// Elements per access: 16 bytes where the pairs and the features that pass come in such pieces (every address and stride
// is a multiple of 16 bytes), else half of that, else single elements.
template <typename T>
int launch_rotary_type(const RotaryArgs& a, bool interleaved, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int rest = a.D - 2 * a.R;
    if (a.R % V == 0 && rest % V == 0) return launch_rotary<T, V>(a, interleaved, st);
    if (a.R % (V / 2) == 0 && rest % (V / 2) == 0) return launch_rotary<T, V / 2>(a, interleaved, st);
    return launch_rotary<T, 1>(a, interleaved, st);
}

int fill(const ca_rotary_desc* d, RotaryArgs* a) {
    if (!d) { set_error("descriptor is NULL"); return CA_ERR_NULL; }
    const int rc = check_seq_dtype(d->dtype);
    if (rc) return rc;
    if (d->dim < 8 || d->dim % 8 || d->dim > 512) { set_error("dim=%d: multiples of 8 up to 512 are supported", d->dim); return CA_ERR_BAD_DESC; }
    if (d->pairs < 1 || 2 * (int64_t)d->pairs > d->dim) { set_error("pairs=%d do not fit into %d features", d->pairs, d->dim); return CA_ERR_BAD_DESC; }
    if (d->axes < 1 || d->axes > CA_MAX_AXES) { set_error("axes=%d: 1 to %d are supported", d->axes, CA_MAX_AXES); return CA_ERR_BAD_DESC; }
    int64_t end = 0;
    for (int i = 0; i < d->axes; ++i) {
        if (d->sections[i] < 0) { set_error("section %d is negative", i); return CA_ERR_BAD_DESC; }
        end += d->sections[i];
        a->ends[i] = (int)(end > d->pairs ? d->pairs : end);
    }
    if (end != d->pairs) { set_error("the sections hold %lld pairs, not %d", (long long)end, d->pairs); return CA_ERR_BAD_DESC; }
    if (d->tokens < 0 || d->batch < 0) { set_error("tokens=%d batch=%d must not be negative", d->tokens, d->batch); return CA_ERR_BAD_DESC; }
    a->tokens = (int64_t)d->tokens * d->batch;
    if (a->tokens > INT32_MAX) { set_error("more than 2^31 - 1 tokens"); return CA_ERR_TOO_LARGE; }
    if (a->tokens && (!d->positions || !d->turns)) { set_error("positions and turns must not be NULL"); return CA_ERR_NULL; }
    a->D = d->dim; a->R = d->pairs; a->axes = d->axes;
    a->pos = d->positions; a->turns = d->turns;
    a->p_axis = d->axis_stride; a->p_token = d->token_stride; a->p_batch = d->batch_stride;
    a->N = d->tokens;
    a->sign = d->inverse ? -1.f : 1.f;
    return CA_OK;
}

RotaryTensor tensor(const ca_seq_view* x, const ca_seq_view* y, int heads, int turn) {
    RotaryTensor t{};
    t.src = x->data; t.s_head = x->head; t.s_token = x->token; t.s_batch = x->batch;
    t.heads = heads; t.turn = turn;
    if (y) { t.dst = y->data; t.d_head = y->head; t.d_token = y->token; t.d_batch = y->batch; }
    return t;
}

int run(RotaryArgs& a, int dtype, int interleaved, cudaStream_t st) {
    for (int i = 0; i < a.nt; ++i) a.total_heads += a.t[i].heads;
    if (a.total_heads > 16384) { set_error("heads=%d: up to 16384 in one call are supported", a.total_heads); return CA_ERR_TOO_LARGE; }
    if (!a.tokens) return CA_OK;
    a.heads_inv = (uint32_t)(((1ULL << 32) + a.total_heads - 1) / a.total_heads);
    // Tokens of a block: as many as leave sixteen blocks for every SM (two rounds), so that the sines fill the threads of a long call,
    // the last round is full and a short call still spreads over the chip (prompts: 63.5 us with rounds of 1.4, 57.7 with two).
    a.per_block = kRotaryTokens;
    while (a.per_block > 1 && a.tokens < 16LL * sm_count() * a.per_block) a.per_block >>= 1;
    if (dtype == CA_F32) return launch_rotary_type<float>(a, interleaved, st);
    if (dtype == CA_BF16) return launch_rotary_type<__nv_bfloat16>(a, interleaved, st);
    return launch_rotary_type<__half>(a, interleaved, st);
}

}  // namespace
}  // namespace ca

using namespace ca;

extern "C" {

int ca_rotary(const ca_rotary_desc* d, const ca_seq_view* x1, const ca_seq_view* y1, int32_t heads1,
              const ca_seq_view* x2, const ca_seq_view* y2, int32_t heads2, void* stream) {
    RotaryArgs a{};
    int rc = fill(d, &a);
    if (rc) return rc;
    if (heads1 < 1 || (x2 && heads2 < 1)) { set_error("heads must be positive"); return CA_ERR_BAD_DESC; }
    if ((rc = check_view(x1, d->dtype, "x1", a.tokens > 0)) || (rc = check_view(y1, d->dtype, "y1", a.tokens > 0))) return rc;
    a.t[a.nt++] = tensor(x1, y1, heads1, 1);
    if (x2) {
        if ((rc = check_view(x2, d->dtype, "x2", a.tokens > 0)) || (rc = check_view(y2, d->dtype, "y2", a.tokens > 0))) return rc;
        a.t[a.nt++] = tensor(x2, y2, heads2, 1);
    }
    return run(a, d->dtype, d->interleaved, as_stream(stream));
}

int ca_rotary_append(const ca_rotary_desc* d, const ca_seq_view* q, const ca_seq_view* q_out, int32_t heads_q,
                     const ca_seq_view* k, const ca_seq_view* v, int32_t heads_kv,
                     const ca_page_view* k_pages, const ca_page_view* v_pages, const ca_pages* pages, void* stream) {
    RotaryArgs a{};
    int rc = fill(d, &a);
    if (rc) return rc;
    if (d->batch != 1) { set_error("packed tokens have batch 1 (got %d)", d->batch); return CA_ERR_BAD_DESC; }
    if (heads_q < 1 || heads_kv < 1) { set_error("heads must be positive"); return CA_ERR_BAD_DESC; }
    if ((rc = check_pages(pages, d->tokens))) return rc;
    if ((rc = check_view(q, d->dtype, "q", a.tokens > 0)) || (rc = check_view(q_out, d->dtype, "q_out", a.tokens > 0)) || (rc = check_view(k, d->dtype, "k", a.tokens > 0)) ||
        (rc = check_view(v, d->dtype, "v", a.tokens > 0)) || (rc = check_page_view(k_pages, d->dtype, "k_pages", a.tokens > 0 && pages->pages)) ||
        (rc = check_page_view(v_pages, d->dtype, "v_pages", a.tokens > 0 && pages->pages)))
        return rc;
    a.t[0] = tensor(q, q_out, heads_q, 1);
    a.t[1] = tensor(k, nullptr, heads_kv, 1);
    a.t[2] = tensor(v, nullptr, heads_kv, 0);
    const ca_page_view* to[2] = {k_pages, v_pages};
    for (int i = 0; i < 2; ++i) {
        RotaryTensor& t = a.t[1 + i];
        t.paged = 1;
        t.dst = to[i]->data; t.d_head = to[i]->head; t.d_token = to[i]->token; t.d_batch = to[i]->page;
    }
    a.nt = 3;
    a.pages = *pages;
    return run(a, d->dtype, d->interleaved, as_stream(stream));
}

}  // extern "C"
