// Shared parts of the operators on token sequences: argument checks, element conversions, which rows and keys a tile of
// the attention holds, and which keys a row sees.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include "common.cuh"
#include "../../include/circatt_b200_tokens.h"

namespace ca {

// ---------------------------------------------------------------- elements
template <typename T> __device__ __forceinline__ float to_float(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// ---------------------------------------------------------------- checks (seq_api.cu)
int check_seq_dtype(int dtype);
int check_view(const ca_seq_view* v, int dtype, const char* name, bool used);         // used: something is read or written there
int check_page_view(const ca_page_view* v, int dtype, const char* name, bool used);
int check_pages(const ca_pages* p, int tokens);

// ---------------------------------------------------------------- attention
// Other scores and masks than the window's.  Kernels that know them are compiled apart (FORM): calls without keep their results to
// the bit, and their time but for the compiler's choices (Float32, before and after: 2 x 4096 tokens, 8 heads of 64 features, forward 206
// and 209 us, dq 275 and 275, dk and dv 354 and 353; 8 chunks of 500 tokens over a cache, 128 features, 3550 and 3491).
struct SeqForm {
    float cap_in, cap_out;          // z = cap_out tanh(cap_in q.k), with scale / cap and cap log2(e); cap_out = 0: no cap
    float poly[6];                  // tanh(|cap_in| x) = x poly(x^2) where that is at most 1: TanhPoly's numbers times powers of |cap_in|
    const float* slopes;            // for each query head, nullable: z -= slope log2(e) |i - j|
    const int4* spans;              // dense: [batch][token], nullable: the token sees x..z, and y..w see it
    const int* prefix;              // paged, [sequence], nullable: tokens below are visible to all of the sequence
};
// What of it a call has.  A kernel is compiled for each kind that needs other arithmetic; kMasks has spans or a prefix only, and all
// of them may have those.
enum FormKind { kNoForm, kMasks, kSlopes, kCap, kCapSlopes };
__host__ __device__ constexpr bool has_cap(int form) { return form >= kCap; }
__host__ __device__ constexpr bool has_slopes(int form) { return form == kSlopes || form == kCapSlopes; }

// A query tile holds consecutive rows R of one key head: row R is query head R % G of the group, token R / G, so that
// the query heads that share a key head share its tiles.
struct SeqArgs {
    int D, Hq, Hkv, G;
    uint32_t g_mul, g_shift;        // R / G = R * g_mul >> g_shift for 0 <= R < 2^31
    int N, B;                       // dense: tokens and batch; paged: packed tokens and 1
    int left, right, sinks;         // left: kNoLeft without a left end
    float scale, scale_log2;        // scale_log2 = scale * log2(e)
    float mag_log2;                 // its magnitude, never 0 (0 * -inf of a masked score would be NaN): the sign goes to q
    const int* lengths;             // dense: nullable; paged: tokens in the cache
    ca_seq_view q, k, v, y, rest, dy, dq, dk, dv;   // rest.data nullable: what rounding took from y
    ca_page_view kp, vp;
    ca_pages pages;                 // table == nullptr: dense
    SeqForm form;
    int kind;                       // of FormKind
    int ranked;                     // Float32: tiles of unequal work, the largest first
    float* lse;                     // [b][key head][R]: log2 of the sum, -inf for rows that see nothing
    float* delta;                   // the same order: dy . y
    int* status;
};
constexpr int kNoLeft = 1 << 30;

// Token of row R.  A division by a number that the compiler does not know costs some forty instructions.
__device__ __forceinline__ int token_of(const SeqArgs& a, int R) { return (int)((uint64_t)(uint32_t)R * a.g_mul >> a.g_shift); }

// The sequence that a tile works on.
struct Seq {
    int b;          // batch index / sequence
    int T;          // its rows' tokens
    int t0;         // first packed token (paged)
    int base;       // position of token 0
    int n;          // tokens that exist: positions 0 .. n-1
};

__device__ __forceinline__ Seq dense_seq(const SeqArgs& a, int b) {
    Seq s{b, a.N, 0, 0, a.N};
    if (a.lengths) s.n = max(0, min(a.N, a.lengths[b]));
    return s;
}

// Finds the sequence that owns row tile `idx` of `rows` rows (tiles numbered sequence by sequence) and leaves the tile's
// number within it in idx; false behind the last tile.  Every lane of a warp calls it together.
__device__ __forceinline__ bool paged_seq(const SeqArgs& a, int rows, int& idx, Seq* s) {
    const int lane = threadIdx.x & 31, S = a.pages.sequences;
    for (int s0 = 0; s0 < S; s0 += 32) {
        const int i = s0 + lane;
        int t0 = 0, T = 0;
        if (i < S) {
            t0 = max(0, min(a.N, a.pages.starts[i]));
            T = max(0, min(a.N, a.pages.starts[i + 1]) - t0);
        }
        const int tiles = (int)(((int64_t)T * a.G + rows - 1) / rows);
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned hit = __ballot_sync(~0u, idx < upto);
        if (hit) {
            const int at = __ffs(hit) - 1;
            s->b = s0 + at;
            s->t0 = __shfl_sync(~0u, t0, at);
            s->T = __shfl_sync(~0u, T, at);
            s->n = max(0, a.pages.lengths[s->b]);
            s->base = s->n - s->T;
            idx -= __shfl_sync(~0u, upto - tiles, at);
            return true;
        }
        idx -= __shfl_sync(~0u, upto, 31);
    }
    return false;
}

// Packed tokens of no sequence (before the first start, behind the last: a call of fixed size that is not full) get zeros.
// `owned`: the tokens of sequences, loaded where a kernel begins and used where it waits for its first copies, so that it
// costs nothing (kernel with one token for each of 64 and of 4 sequences: 181.5 and 13.7 us, 182.4 and 13.8 without).
__device__ __forceinline__ int2 owned_tokens(const SeqArgs& a) { return make_int2(a.pages.starts[0], a.pages.starts[a.pages.sequences]); }

// `thread` of `threads` in each CTA; the CTAs of key head h share the work.
template <typename T>
__device__ __forceinline__ void clear_unowned(const SeqArgs& a, int2 owned, int h, int thread, int threads) {
    const int head = max(0, min(a.N, owned.x)), tail = max(head, min(a.N, owned.y));
    const int count = head + a.N - tail;
    if (!count) return;
    constexpr int V = 16 / sizeof(T);
    const int pieces = a.D / V;
    const int64_t items = (int64_t)count * a.G * pieces;
    for (int64_t i = (int64_t)blockIdx.x * threads + thread; i < items; i += (int64_t)gridDim.x * threads) {
        const int64_t r = i / pieces, t = r / a.G;
        T* y = (T*)a.y.data + (h * a.G + r % a.G) * a.y.head + (t < head ? t : tail + t - head) * a.y.token;
        reinterpret_cast<uint4*>(y)[i % pieces] = make_uint4(0, 0, 0, 0);
    }
}

// Most row tiles that the packed tokens of S sequences can have.
static inline int64_t paged_tiles(int64_t tokens, int64_t G, int64_t S, int64_t rows) {
    const int64_t full = tokens * G / rows + S;
    return full < tokens * G ? full : tokens * G;
}

// Tiles of `keys` keys that a tile of queries at positions p_lo .. p_hi has to look at: first those of the first tokens
// that end before the window's, then the window's.
struct KeyTiles {
    int first;      // tiles of first tokens, from key 0
    int lo;         // first key of the window's first tile
    int count;      // all tiles
    __device__ __forceinline__ int key(int i, int keys) const { return i < first ? i * keys : lo + (i - first) * keys; }
};

// Keys that can exist: a cache holds no more than its table has places for, whatever the length says.
__device__ __forceinline__ int key_limit(const SeqArgs& a, const Seq& s) {
    return a.pages.table ? (int)min((int64_t)min(s.n, 1 << 30), (int64_t)a.pages.width * a.pages.page) : s.n;
}

// The keys from lo to hi, and of those below `sinks` the ones up to hi.
struct Reach { int lo, hi; };

// What the token at `pos` sees.  Both ends never fall from one token to the next (documents and groups follow one another), so
// that a tile's first and last row bound what it sees.
template <int FORM>
__device__ __forceinline__ Reach reach(const SeqArgs& a, const Seq& s, int pos) {
    Reach r{pos - a.left, (int)min((int64_t)INT32_MAX, (int64_t)pos + a.right)};
    if constexpr (FORM) {
        if (a.form.spans) {
            const int4 w = a.form.spans[(int64_t)s.b * a.N + max(0, min(pos, a.N - 1))];
            r.lo = max(r.lo, w.x);
            r.hi = w.z;
        } else if (a.form.prefix) {
            r.hi = max(r.hi, max(0, a.form.prefix[s.b]) - 1);          // the lowest Int32 less 1 would be the highest
        }
    }
    return r;
}
// The same for the bounds of tiles: always with the token itself, whatever the spans hold, so that the tiles of neighbouring
// rows leave no gap.
template <int FORM>
__device__ __forceinline__ Reach tile_reach(const SeqArgs& a, const Seq& s, int pos) {
    Reach r = reach<FORM>(a, s, pos);
    if (FORM) r.lo = min(r.lo, pos), r.hi = max(r.hi, pos);
    return r;
}
// Queries from lo to hi see key j.
__device__ __forceinline__ Reach seen_by(const SeqArgs& a, const Seq& s, int j) {
    const int4 w = a.form.spans[(int64_t)s.b * a.N + max(0, min(j, a.N - 1))];
    return Reach{w.y, min(w.w, j + a.left)};
}

// Padding, which sees nothing and which nothing sees: whatever it holds, it counts as zeros.  `mixed`: there may be some among
// the tokens from..upto, which are not all of one document.
template <int FORM>
__device__ __forceinline__ bool padding(const SeqArgs& a, const Seq& s, int j) {
    if (!FORM || !a.form.spans) return false;
    const int4 w = a.form.spans[(int64_t)s.b * a.N + max(0, min(j, a.N - 1))];
    return w.w < w.y;
}
template <int FORM>
__device__ __forceinline__ bool mixed(const SeqArgs& a, const Seq& s, int from, int upto) {
    if (!FORM || !a.form.spans) return false;
    const int4 w = a.form.spans[(int64_t)s.b * a.N + max(0, min(upto, s.n - 1))];
    return w.x > from || w.w < w.y;
}

// Tiles from..upto that lie between the begin of the last row's document and that row are known to be of one document without
// a look at the spans.
template <int FORM>
__device__ __forceinline__ int document_of(const SeqArgs& a, const Seq& s, int last) {
    return FORM && a.form.spans && last >= 0 ? a.form.spans[(int64_t)s.b * a.N + min(last, a.N - 1)].x : 0;
}

// Keys that the rows from..to - 1 together see: the work of their tile.
template <int FORM>
__device__ __forceinline__ int row_work(const SeqArgs& a, const Seq& s, int from, int to) {
    const int lo = from / a.G, hi = min(s.n - 1, (min(to, s.T * a.G) - 1) / a.G);
    return hi < lo ? 0 : tile_reach<FORM>(a, s, hi).hi - max(0, tile_reach<FORM>(a, s, lo).lo);
}

// Documents make tiles of unequal work, and those are best begun with the largest (packed training: dk and dv 342 -> 249 us, forward
// 259 -> 234).  Each block finds the tile of its rank by itself: runs of neighbouring tiles, at most 128 so that this stays short
// (512 of them took 5 us a block), are ordered by `work(first, last)`, for equal work by number; a last run that is shorter comes
// last.  It costs a block 1.7 us, which dq with its many and even tiles does not get back (263 -> 289 us).
// The block's threads call it together; `counts` has room for 128 numbers, and is free again behind it.
template <typename Work>
__device__ __forceinline__ int ranked_tile(int tiles, int rank, int* counts, int* result, Work work) {
    const int length = (tiles + 127) / 128, runs = (tiles + length - 1) / length, t = threadIdx.x;
    if (t < 128) counts[t] = t >= runs ? -2 : (t + 1) * length > tiles ? -1 : max(0, work(t * length, (t + 1) * length - 1));
    __syncthreads();
    if (t < runs) {
        const int own = counts[t];
        int before = 0;
        for (int i = 0; i < 128; i += 4) {
            const int4 c = *reinterpret_cast<const int4*>(counts + i);
            before += (c.x > own || (c.x == own && i < t)) + (c.y > own || (c.y == own && i + 1 < t)) + (c.z > own || (c.z == own && i + 2 < t)) +
                      (c.w > own || (c.w == own && i + 3 < t));
        }
        if (before == rank / length) *result = t * length + rank % length;
    }
    __syncthreads();
    return *result;
}
// The block's rank, head and sequence, with the heads and sequences innermost, so that the largest tiles of all come first.
struct Place { int x, h, b; };
__device__ __forceinline__ Place place_by_rank() {
    const uint32_t id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z), all = gridDim.y * gridDim.z;
    return Place{(int)(id / all), (int)(id % all % gridDim.y), (int)(id % all / gridDim.y)};
}

template <int FORM = kNoForm>
__device__ __forceinline__ KeyTiles key_tiles(const SeqArgs& a, const Seq& s, int p_lo, int p_hi, int keys) {
    KeyTiles k;
    p_lo = max(p_lo, 0);
    p_hi = min(p_hi, s.n - 1);
    if (p_hi < p_lo) return KeyTiles{0, 0, 0};
    const int limit = key_limit(a, s);
    const int lo = max(0, tile_reach<FORM>(a, s, p_lo).lo);                                  // left <= 2^30
    const int hi = (int)min((int64_t)limit, (int64_t)tile_reach<FORM>(a, s, p_hi).hi + 1);  // > lo unless the table ends before the window
    // A window that begins behind the table has no tile: rounded down to one it would be a tile that no row sees, whose copies nobody
    // waits for.
    k.lo = lo < hi ? lo / keys * keys : hi;
    k.first = (min(a.sinks, k.lo) + keys - 1) / keys;
    k.count = k.first + (lo < hi ? (hi - k.lo + keys - 1) / keys : 0);
    return k;
}

// Whether the query at `pos`, which reaches r, sees key j.
__device__ __forceinline__ bool sees(const SeqArgs& a, int n, int pos, Reach r, int j) {
    return pos >= 0 && pos < n && j < n && j <= r.hi && (j >= r.lo || j < a.sinks);
}
// Whether the query at `pos` sees key j.
__device__ __forceinline__ bool sees(const SeqArgs& a, int n, int pos, int j) {
    return pos >= 0 && pos < n && j < n && j - pos <= a.right && (pos - j <= a.left || j < a.sinks);
}

// Page of key j of sequence b, or -1.
__device__ __forceinline__ int page_of(const SeqArgs& a, int b, int j) {
    const int c = j / a.pages.page;
    if (c >= a.pages.width) return -1;
    const int p = a.pages.table[c + (int64_t)a.pages.width * b];
    return p < a.pages.pages ? p : -1;
}

// ---------------------------------------------------------------- scores with a cap and a slope
// tanh(x) / x on |x| <= 1 as a polynomial in x^2 that minimises the largest relative error (Lawson's iteration): 6.9e-6 with
// degree 4, for bfloat16 weights (scores of 40 are off by 3e-4, a seventh of the weights' rounding); 6.1e-7 with 5 for half; 6.8e-8
// with 6 for Float32 (of the coefficients as they are here, in Float32).
template <int DEGREE> struct TanhPoly;
template <> struct TanhPoly<4> {
    static __host__ __device__ constexpr float at(int i) {
        constexpr float c[5] = {0.999993086f, -0.332980663f, 0.130368114f, -0.0448175557f, 0.00903642457f};
        return c[i];
    }
};
template <> struct TanhPoly<5> {
    static __host__ __device__ constexpr float at(int i) {
        constexpr float c[6] = {0.999999404f, -0.333290428f, 0.132814333f, -0.0516056754f, 0.0167431161f, -0.00306706037f};
        return c[i];
    }
};
template <> struct TanhPoly<6> {
    static __host__ __device__ constexpr float at(int i) {
        constexpr float c[7] = {0.99999994f, -0.333328396f, 0.13325204f, -0.0534570292f, 0.0202899817f, -0.00620337948f, 0.00104102271f};
        return c[i];
    }
};
// tanh(x) = 1 - 2 / (1 + e^2x): an absolute error of 10^-7 or so, which is a relative one where |x| > 1.
__device__ __forceinline__ float tanh_far(float x) { return 1.f - __fdividef(2.f, 1.f + fast_exp2(x * (2.f * kLog2e))); }
__device__ __forceinline__ float tanh_any(float x) {
    const float u = x * x;
    float p = TanhPoly<6>::at(6);
#pragma unroll
    for (int i = 5; i >= 0; --i) p = fmaf(p, u, TanhPoly<6>::at(i));
    return fabsf(x) <= 1.f ? p * x : tanh_far(x);          // what is not a number stays so
}
// Of query head `head`, in units of log2(e).
__device__ __forceinline__ float slope_of(const SeqArgs& a, int head) { return a.form.slopes ? a.form.slopes[head] * kLog2e : 0.f; }
// A score in units of log2(e), from q.k, less `minus`; slope in those units too, `inner`: the derivative of the cap.
template <int FORM>
__device__ __forceinline__ float formed_score(const SeqArgs& a, float dot, float slope, int distance, float minus, float& inner) {
    inner = 1.f;
    if (!has_cap(FORM) && !has_slopes(FORM)) return fmaf(dot, a.scale_log2, -minus);         // as without a form, to the bit
    float z = dot * a.scale_log2;
    if (has_cap(FORM)) {
        const float t = tanh_any(dot * a.form.cap_in);
        z = a.form.cap_out * t;
        inner = fmaf(-t, t, 1.f);
    }
    return has_slopes(FORM) ? fmaf(-slope, fabsf((float)distance), z) - minus : z - minus;
}

// How the backward deals out the queries of key tiles that hold first tokens: those tiles have every later query, an ordinary one
// those of its window.
struct Dealt {
    int tiles, segments;            // the first key tiles, and the CTAs for each
};
static inline Dealt deal_first_tokens(const SeqArgs& a, int tile) {
    // Pieces of about an ordinary tile's work, as long as they are few: each leaves a Float32 part of dk and dv (128 KB at 128
    // features).  Seven CTAs for every SM even out the work; many first tokens, heads or sequences fill the chip without.  2 x 8192
    // tokens, 8 heads of 64 features, window 256, 4096 first tokens, dk and dv: 334 us with 2 pieces, 754 with 22 (640 MB more).
    constexpr int64_t kMost = 64, kParts = 1024;
    const int64_t all = ((int64_t)a.N + tile - 1) / tile, window = ((int64_t)a.left + a.right + 2 * tile - 1) / tile;
    const int64_t tiles = ((int64_t)(a.sinks < a.N ? a.sinks : a.N) + tile - 1) / tile;
    int64_t segments = (all + window - 1) / window;
    if (segments > kMost) segments = kMost;
    if (tiles && segments > kParts / (tiles * a.Hkv * a.B)) segments = kParts / (tiles * a.Hkv * a.B);
    return tiles && segments > 1 ? Dealt{(int)tiles, (int)segments} : Dealt{0, 1};
}

// seq_fma.cu: Float32 on the FMA pipe
int fma_fwd(const SeqArgs& a, cudaStream_t st);               // dense or paged
size_t fma_bwd_parts(const SeqArgs& a);
int fma_bwd(const SeqArgs& a, float* parts, cudaStream_t st);

}  // namespace ca
