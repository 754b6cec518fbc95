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

__device__ __forceinline__ KeyTiles key_tiles(const SeqArgs& a, const Seq& s, int p_lo, int p_hi, int keys) {
    KeyTiles k;
    p_lo = max(p_lo, 0);
    p_hi = min(p_hi, s.n - 1);
    if (p_hi < p_lo) return KeyTiles{0, 0, 0};
    const int limit = key_limit(a, s);
    const int lo = max(0, p_lo - a.left);                                  // left <= 2^30
    const int hi = (int)min((int64_t)limit, (int64_t)p_hi + a.right + 1);  // > lo unless the table ends before the window
    // A window that begins behind the table has no tile: rounded down to one it would be a tile that no row sees, whose copies nobody
    // waits for.
    k.lo = lo < hi ? lo / keys * keys : hi;
    k.first = (min(a.sinks, k.lo) + keys - 1) / keys;
    k.count = k.first + (lo < hi ? (hi - k.lo + keys - 1) / keys : 0);
    return k;
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
