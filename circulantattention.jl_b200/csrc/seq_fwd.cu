// Attention on token sequences, forward, on the tensor cores (tcgen05): dense tensors and a paged cache, 16-bit types.
//
// A CTA takes tiles of 128 query rows of one key head and walks the tiles of 128 keys that they see, with a running maximum
// and sum per row.  Scores of a tile come into tensor memory (128 lanes = rows, 128 columns = keys); the thread that owns the
// row reads them, turns them into weights, and writes those back over the scores as 16-bit pairs, from where the second
// product takes them as its A operand: the weights never see shared memory.
//
// Roles: two groups of four warps do the softmax, one warp copies keys and values by TMA into a ring of tiles, one warp
// issues the products.  The two groups are two streams that share the tensor cores: while one turns its scores into weights,
// the products of the other run.  With PAIR the streams are two row tiles that share every key tile (half the copies); without,
// they take the even and the odd key tiles of one row tile and are joined at the end (few rows).
//
// The accumulator is rescaled only where a row's maximum grew by more than 2^8 since its reference: the weights stay below
// 2^8, and the products and sums are held in Float32.  Weights are rounded to the tensors' type before their product, once more
// than the result itself: errors are 1.15 to 1.6 of those of a plain implementation that keeps them in Float32.
//
// Bound: the exponentials and the products, 2048 cycles each for a pair of 128 x 128 tiles at 128 features; a pair takes about
// 3300 in the steady state, since a row's chain (scores, maximum, exponentials, weights) leaves gaps that two streams do not
// fill.  Measured: 65536 tokens, window 4096, 16 query and 2 key heads 2.03 ms (1.05 PFLOP/s of visible pairs; a
// large matrix product has 1.62 in a burst and keeps up 1.37; 1.99 to 2.14 ms by box, at the power cap); 2 x 16384 tokens, window 1024, 16 and 4 heads 415 us.
#include "seq_umma.cuh"

#include <limits.h>

namespace ca {
namespace {

// Two warpgroups of softmax, a warp that copies and one that issues the products.
constexpr int kThreads = 320, kSoftmaxWarps = 8;

template <int DM> constexpr uint32_t kTileBytes = 128 * DM * 2;
template <int DM> constexpr int kSlots = DM == 128 ? 5 : 8;
template <int DM> constexpr size_t kFwdSmem = (size_t)(2 + kSlots<DM>) * kTileBytes<DM> + 1024;

struct FwdMaps {
    CUtensorMap k, v, q, y, rest;
    int rows;           // q, y and rest move by tiles of rows (maps), else by threads
    int box;            // paged: keys of a box
    int* timeouts;
};

// A stream's tiles: those of first tokens below `first`, then from..upto, in steps of one (PAIR) or two.
struct Stream {
    int lo, hi;             // positions of its rows that exist; lo > hi: none
    int first, from, upto, step;
    int begin_key, end_key;     // its rows' windows together
    // Whether any row sees a key of the half tile from `key0`.  What a tile costs is its exponentials, so halves outside the
    // windows (the tiles at their ends, a few first tokens) are left out.
    __device__ __forceinline__ bool sees_half(const SeqArgs& a, int key0) const { return key0 <= end_key && (key0 + 63 >= begin_key || key0 < a.sinks); }
    __device__ __forceinline__ bool takes(int i) const { return step == 2 ? (i & 1) == (from & 1) && i <= upto : i < first || (i >= from && i <= upto); }
    __device__ __forceinline__ int begin() const { return first > 0 ? 0 : from; }
    __device__ __forceinline__ int next(int i) const {
        i += step;
        return i >= first && i < from ? from : i;
    }
};

template <bool PAIR>
__device__ __forceinline__ Stream stream_of(const SeqArgs& a, const Seq& s, const KeyTiles& kt, int u, int r, int rows) {
    Stream t;
    t.lo = max(0, s.base + r / a.G);
    t.hi = r < rows ? min(s.n - 1, s.base + (min(r + 128, rows) - 1) / a.G) : -1;
    t.begin_key = max(0, t.lo - a.left);
    t.end_key = (int)min((int64_t)key_limit(a, s) - 1, (int64_t)t.hi + a.right);
    if (!PAIR) {
        t.first = 0;
        t.from = u;
        t.upto = kt.count - 1;
        t.step = 2;
        return t;
    }
    t.step = 1;
    if (t.hi < t.lo) {
        t.first = 0;
        t.from = 0;
        t.upto = -1;
        return t;
    }
    // the window's tiles begin at kt.lo; those of first tokens lie before it, and beyond it only up to the window
    const int known = min(a.sinks, key_limit(a, s)), firsts = kt.first + (known > kt.lo ? (known - kt.lo + 127) / 128 : 0);
    if (t.end_key < t.begin_key) {          // the table ends before these rows' windows: first tokens only
        t.first = t.from = firsts;
        t.upto = firsts - 1;
        return t;
    }
    t.from = kt.first + max(0, t.begin_key - kt.lo) / 128;
    t.upto = t.end_key >= kt.lo ? kt.first + (t.end_key - kt.lo) / 128 : kt.first - 1;
    t.first = max(kt.first, min(min(t.from, t.upto + 1), firsts));
    return t;
}

template <typename T, int DM, bool PAIR, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) umma_fwd_kernel(const __grid_constant__ SeqArgs a, const __grid_constant__ FwdMaps maps) {
    constexpr int S = kSlots<DM>;
    constexpr uint32_t TILE = kTileBytes<DM>;
    constexpr uint32_t IDESC_S = instr_desc(kIsBf16<T>, 128, false), IDESC_O = instr_desc(kIsBf16<T>, DM, true);
    extern __shared__ char raw[];
    __shared__ uint64_t kv_full[S], kv_empty[S], q_full[2], s_full[2], p_full[2][2], o_full[2], drained;
    __shared__ uint32_t tmem_slot, valid[S];
    __shared__ int stop_flag;
    __shared__ float merge_m[128], merge_l[128];
    volatile int* stop = &stop_flag;

    const uint32_t raw_at = smem_u32(raw), base_at = (raw_at + 1023) & ~1023u;
    char* const smem = raw + (base_at - raw_at);
    const uint32_t q_at = base_at, kv_at = base_at + 2 * TILE;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    int tile = (int)(gridDim.x - 1 - blockIdx.x);       // the last rows see the most keys: first
    int2 owned;
    Seq s;
    if (PAGED) {
        owned = owned_tokens(a);
        if (!paged_seq(a, PAIR ? 256 : 128, tile, &s)) {
            if (tid < 32 * kSoftmaxWarps) clear_unowned<T>(a, owned, h, tid, 32 * kSoftmaxWarps);
            return;
        }
    } else {
        s = dense_seq(a, blockIdx.z);
    }
    const int rows = s.T * a.G, R0 = tile * (PAIR ? 256 : 128);
    const int p_lo = max(0, s.base + R0 / a.G), p_hi = min(s.n - 1, s.base + (min(R0 + (PAIR ? 256 : 128), rows) - 1) / a.G);
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, 128);

    // Which key tiles a stream takes: with PAIR both see nearly the same, but each leaves out what all of its rows are blind to.
    const Stream st0 = stream_of<PAIR>(a, s, kt, 0, R0, rows), st1 = stream_of<PAIR>(a, s, kt, 1, PAIR ? R0 + 128 : R0, rows);

    if (warp == 8 && lane == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int u = 0; u < 2; ++u) {
            mbar_init(&q_full[u], maps.rows ? 1 : PAIR ? 4 : 8);
            mbar_init(&s_full[u], 1);
            mbar_init(&p_full[u][0], 4);
            mbar_init(&p_full[u][1], 4);
            mbar_init(&o_full[u], 1);
        }
        mbar_init(&drained, 1);
        stop_flag = 0;
        mbar_fence_init();
        fence_async_smem();
        if (maps.rows) {                                                   // on their way while the rest is set up
            for (int u = 0; u < (PAIR ? 2 : 1); ++u) {
                if (R0 + 128 * u >= rows) break;
                mbar_arrive_expect_tx(smem_u32(&q_full[u]), TILE);
#pragma unroll
                for (int p = 0; p < DM / 64; ++p)
                    tma_load_4d(q_at + u * TILE + p * kPanel, &maps.q, 64 * p, h * a.G, s.t0 + (R0 + 128 * u) / a.G, PAGED ? 0 : s.b, smem_u32(&q_full[u]));
            }
        }
        prefetch_map(&maps.k);
        prefetch_map(&maps.v);
    }
    if (warp == 9) tmem_alloc(smem_u32(&tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    // Scores of both streams, then their accumulators.  At 64 features there is room for weights beside the scores; at 128 they
    // overlay them, which needs the next scores to be written after the product with the weights has read them: products of
    // one shape (both 128 x 128 x 16 there) are carried out in the order of their issue.
    const uint32_t s_col = tmem, o_col = tmem + 256, p_col = DM == 64 ? tmem + 384 : s_col, p_step = DM == 64 ? 64 : 128;

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax: thread = row
        const int u = warp >> 2, r = tid & 127;
        const Stream st = u ? st1 : st0;
        const int R = R0 + (PAIR ? 128 * u : 0) + r;
        const int pos = s.base + token_of(a, R);
        const bool have = R < rows, live = have && pos >= 0 && pos < s.n;
        if (!maps.rows) {
            const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;        // scores use the scale's magnitude
            // rows of the tile that exist: those of positions 0 .. n - 1
            const int tile0 = R - r;
            const int from = (int)min((int64_t)128, max((int64_t)0, -(int64_t)s.base * a.G - tile0));
            const int to = (int)min((int64_t)rows, ((int64_t)s.n - s.base) * a.G) - tile0;
            auto row = [&](int rr) { return seq_row<T>(a.q, a, s, h, min(tile0 + rr, rows - 1)); };
            constexpr int THREADS = PAIR ? 128 : 256;
            const int t = PAIR ? r : tid;
            uint4 w[TileCopy<DM, THREADS>::kCount];
            fetch_tile<T, DM, THREADS>(w, row, from, to, a.D, t);
#pragma unroll
            for (int i = 0; i < TileCopy<DM, THREADS>::kCount; ++i) { w[i].x ^= sign; w[i].y ^= sign; w[i].z ^= sign; w[i].w ^= sign; }
            put_tile<DM, THREADS>(smem + (PAIR ? u : 0) * TILE, w, t);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[PAIR ? u : 0]));
        }
        const uint32_t lane_off = (uint32_t)(warp & 3) << 21;              // lane 32 * (warp % 4) in bits 16..
        const uint32_t S_at = s_col + u * 128 + lane_off, P_at = p_col + u * p_step + lane_off, O_at = o_col + u * DM + lane_off;
        const float sl2 = a.mag_log2;
        const int c_lo = p_lo - a.left, c_hi = min(p_hi + a.right, s.n - 1);   // keys that any row of the CTA sees (or < sinks)
        // tiles from in_lo (or below in_sink) to in_hi need no mask
        const bool whole = st.lo == s.base + (R - r) / a.G && st.hi == s.base + (min(R - r + 128, rows) - 1) / a.G;
        const int in_hi = whole ? min(st.lo + a.right, s.n - 1) - 127 : INT_MIN, in_lo = st.hi - a.left, in_sink = a.sinks - 127;
        float m = -INFINITY, l = 0.f;
        int done = 0;
        bool ok = true;
        if (PAGED) clear_unowned<T>(a, owned, h, tid, 32 * kSoftmaxWarps);
        for (int i = st.begin(); i <= st.upto; i = st.next(i)) {
            const int key0 = kt.key(i, 128), vslot = (2 * i + 1) % S;
            const uint32_t vpar = ((2 * i + 1) / S) & 1;
            if (!warp_wait(smem_u32(&s_full[u]), done & 1, stop)) { ok = false; break; }
            fence_after();
            uint32_t there = 0xff;
            if (PAGED) {                                                   // which pages exist is known when their copy has landed
                if (!warp_wait(smem_u32(&kv_full[vslot]), vpar, stop)) { ok = false; break; }
                there = *(volatile uint32_t*)&valid[vslot];
            }
            const int far = key0 + 127;
            const bool edge = !(key0 <= in_hi && (key0 >= in_lo || key0 < in_sink) && there == 0xff);
            const int hi = live ? min(pos + a.right, s.n - 1) - key0 : -1, lo = pos - a.left - key0, sk = a.sinks - key0;
            auto scores = [&](int g, uint32_t* x) {                        // the columns 64 g .. 64 g + 63
                tmem_ld32(S_at + 64 * g, x);
                tmem_ld32(S_at + 64 * g + 32, x + 32);
                tmem_wait_ld();
                settled32(x);
                settled32(x + 32);
            };
            // The same for the maximum: -inf where the row does not see the key, written back for the exponentials
            auto masked_scores = [&](int g, uint32_t* x) {
                scores(g, x);
                if (edge) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int at = 64 * g + 32 * q;
                        uint32_t mk = seen_bits(lo - at, hi - at, sk - at);
                        if (PAGED) mk &= ((there >> (at / 16)) & 1 ? 0xffffu : 0u) | ((there >> (at / 16 + 1)) & 1 ? 0xffff0000u : 0u);
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[32 * q + c] = (mk >> c) & 1 ? x[32 * q + c] : 0xff800000u;
                        tmem_st32(S_at + at, x + 32 * q);
                    }
                }
            };
            // values that no row sees may be anything (a page that was freed, tokens behind the length): zeros
            if (!((key0 >= c_lo || far < a.sinks) && far <= c_hi && there == 0xff)) {
                if (!PAGED && !warp_wait(smem_u32(&kv_full[vslot]), vpar, stop)) { ok = false; break; }
                const int j = key0 + r;
                if (!(j <= c_hi && (j >= c_lo || j < a.sinks) && (there >> (r >> 4) & 1))) {
#pragma unroll 1
                    for (int p = 0; p < DM / 64; ++p)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            *reinterpret_cast<uint4*>(smem + (2 + vslot) * TILE + p * kPanel + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            float mx = -INFINITY;
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                if (!st.sees_half(a, key0 + 64 * g)) continue;
                uint32_t x[64];
                masked_scores(g, x);
                float top[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = fmaxf(fmaxf(top[e], __uint_as_float(x[c + e])), __uint_as_float(x[c + 4 + e]));
                mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            }
            tmem_wait_st();
            mx *= sl2;
            float f = 1.f;
            const bool grew = mx > m + 8.f;                                // also from -inf
            if (grew) {
                f = fast_exp2(m - mx);
                m = mx;
            }
            if (done && __any_sync(~0u, grew)) {
                // the scores came after the previous weighted sum, which is therefore complete
#pragma unroll 1
                for (int c = 0; c < DM; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(O_at + c, o);
                    tmem_wait_ld();
                    settled32(o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st32(O_at + c, o);
                }
            }
            const float ref = m == -INFINITY ? 0.f : m;                    // a row that has seen nothing yet
            const f32x2 sc2 = pack2(sl2, sl2), ref2 = pack2(-ref, -ref);
            f32x2 sum2 = pack2(l * f, 0.f);
#pragma unroll 1
            for (int g = 0; g < 2; ++g) {
                if (!st.sees_half(a, key0 + 64 * g)) continue;
                uint32_t x[64], w[32];
                scores(g, x);
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1])), sc2, ref2), e0, e1);
                    // The exponential unit and the tensor pipe take the same 2048 cycles a pair of tiles; a quarter of the
                    // exponentials as polynomials: 443 -> 418 us for a sequence of 16384 (an eighth: 431, a half: 430).
                    if (c % 4 == 3) {
                        unpack2(exp2_fma<T>(e0, e1), e0, e1);
                    } else {
                        e0 = fast_exp2(e0);
                        e1 = fast_exp2(e1);
                    }
                    sum2 = add2(sum2, pack2(e0, e1));
                    w[c] = pack16<T>(e0, e1);
                }
                tmem_st32(P_at + 32 * g, w);                               // at 128 features over scores that this warp has read twice
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[u][g]));       // the product with the first half may start
            }
            float a0, a1;
            unpack2(sum2, a0, a1);
            l = a0 + a1;
            ++done;
        }
        if (done && ok) ok = warp_wait(smem_u32(&o_full[u]), 0, stop);
        // without key tiles nothing has waited for the queries, whose place the results take
        if (!done && maps.rows && (PAIR || u == 0) && R - r < rows) ok = warp_wait(smem_u32(&q_full[PAIR ? u : 0]), 0, stop) && ok;
        fence_after();

        // ------------------------------------------------------------ results
        float f0 = 1.f, f1 = 0.f;
        float* const other = reinterpret_cast<float*>(smem + 2 * TILE);    // [column][row] of the odd stream, in the ring's place
        const bool keep_rest = !PAGED && a.rest.data;
        if (!PAIR || keep_rest) group_sync<256>(1);                        // both streams are through with the ring
        if (!PAIR) {
            if (u == 1) {
                merge_m[r] = m;
                merge_l[r] = l;
                if (done && ok) {
#pragma unroll 1
                    for (int c = 0; c < DM; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(O_at + c, o);
                        tmem_wait_ld();
                        settled32(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) other[(c + e) * 128 + r] = __uint_as_float(o[e]);
                    }
                }
            }
            group_sync<256>(1);
            const float m1 = merge_m[r], l1 = merge_l[r], M = fmaxf(m, m1), ref = M == -INFINITY ? 0.f : M;
            f0 = fast_exp2(m - ref);
            f1 = fast_exp2(m1 - ref);
            l = l * f0 + l1 * f1;
            m = M;
        }
        if (PAIR || u == 0) {
            float inv = l > 0.f ? 1.f / l : 0.f;
            if (!ok || *stop) inv = __int_as_float(0x7fffffff);            // a wait ran out: NaN, never a wrong number
            // Rows that see nothing are zeros by choice, not by their weights: 0 * inf of a value that other rows see is not a number.
            const bool none = !done || l == 0.f, both = !PAIR && kt.count > 1 && !none;
            if (!PAGED && a.lse && have) a.lse[((int64_t)s.b * a.Hkv + h) * rows + R] = l > 0.f ? m + log2f(l) : -INFINITY;
            const float w0 = f0 * inv, w1 = f1 * inv;
            // y goes to the queries' place (their last scores are done), what rounding took to a slot of the ring
            const int tile0 = R - r;
            char *const out = smem + (PAIR ? u : 0) * TILE, *const out_rest = smem + (2 + (PAIR ? u : 2)) * TILE;
#pragma unroll 1
            for (int c = 0; c < DM; c += 32) {
                uint32_t o[32];
                tmem_ld32(O_at + c, o);
                tmem_wait_ld();
                settled32(o);
                float y[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) y[e] = __uint_as_float(o[e]) * w0;
                if (none) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = 0.f * inv;
                }
                if (both) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = fmaf(other[(c + e) * 128 + r], w1, y[e]);
                }
                put_row32<T>(out, r, c, y);
                if (keep_rest) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] -= to_float(from_float<T>(y[e]));
                    put_row32<T>(out_rest, r, c, y);
                }
            }
            fence_async_smem();
            group_sync<128>(2 + u);
            // by maps, which leave out tokens behind the tensor's; a cache's packed rows go on with the next sequence
            if (maps.rows && (!PAGED || tile0 + 128 <= rows)) {
                if (r == 0 && tile0 < rows) {
                    const int token = s.t0 + tile0 / a.G, b = PAGED ? 0 : s.b;
#pragma unroll
                    for (int p = 0; p < DM / 64; ++p) {
                        tma_store_4d(&maps.y, smem_u32(out) + p * kPanel, 64 * p, h * a.G, token, b);
                        if (keep_rest) tma_store_4d(&maps.rest, smem_u32(out_rest) + p * kPanel, 64 * p, h * a.G, token, b);
                    }
                    tma_stores_read();
                }
            } else {
                auto row = [&](const ca_seq_view& v) { return [&](int rr) { return seq_row<T>(v, a, s, h, max(tile0 + rr, 0)); }; };
                store_tile<T, DM, 128>(out, row(a.y), rows - tile0, a.D, r);
                if (keep_rest) store_tile<T, DM, 128>(out_rest, row(a.rest), rows - tile0, a.D, r);
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------ copies
        int issued = 0;
        if (!PAGED) {
            if (lane == 0) {
                for (; issued < 2 * kt.count; ++issued) {
                    const int slot = issued % S;
                    if (!wait_or_stop(smem_u32(&kv_empty[slot]), ((issued / S) & 1) ^ 1, stop)) break;
                    const uint32_t bar = smem_u32(&kv_full[slot]), dst = kv_at + slot * TILE;
                    mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
                    for (int p = 0; p < DM / 64; ++p)
                        tma_load_4d(dst + p * kPanel, issued & 1 ? &maps.v : &maps.k, 64 * p, kt.key(issued >> 1, 128), h, s.b, bar);
                }
            }
        } else {
            const int box = maps.box, chunks = 128 / box;
            bool ok = true;
            for (int i = 0; i < kt.count && ok; ++i) {
                const int j = kt.key(i, 128) + lane * box;
                const int page = lane < chunks && j < s.n ? page_of(a, s.b, j) : -1;
                const unsigned has = __ballot_sync(~0u, page >= 0);
                uint32_t bits = 0;                                         // per 16 keys
                for (int c = 0; c < 8; ++c) bits |= (has >> (c * 16 / box) & 1) << c;
                for (int kv = 0; kv < 2; ++kv, ++issued) {
                    const int slot = issued % S;
                    int go = 1;
                    if (lane == 0) go = wait_or_stop(smem_u32(&kv_empty[slot]), ((issued / S) & 1) ^ 1, stop);
                    if (!__shfl_sync(~0u, go, 0)) { ok = false; break; }
                    const uint32_t bar = smem_u32(&kv_full[slot]), dst = kv_at + slot * TILE;
                    if (lane == 0) {
                        *(volatile uint32_t*)&valid[slot] = bits;
                        mbar_arrive_expect_tx(bar, (uint32_t)__popc(has) * box * DM * 2);
                    }
                    __syncwarp();
                    if (page >= 0) {
#pragma unroll
                        for (int p = 0; p < DM / 64; ++p)
                            tma_load_4d(dst + p * kPanel + lane * box * 128, kv ? &maps.v : &maps.k, 64 * p, j % a.pages.page, h, page, bar);
                    }
                }
            }
        }
        if (maps.rows && lane == 0)                                        // also where no key tile waits for them
            for (int u = 0; u < (PAIR ? 2 : 1) && R0 + 128 * u < rows; ++u) mbar_wait(smem_u32(&q_full[u]), 0, 1u << 12);
        if (lane == 0)                                                     // copies in flight land before the memory goes away
            for (int i = max(0, issued - S); i < issued; ++i) mbar_wait(smem_u32(&kv_full[i % S]), (i / S) & 1, 1u << 12);
    } else if (warp == 9) {
        // ------------------------------------------------------------ products: the warp in step, one lane issues
        const uint32_t lead = elect_one();
        const uint64_t q_desc = desc_features(q_at), k_desc = desc_features(kv_at), v_desc = desc_rows(kv_at);
        bool ok = true;
        uint32_t scored = 0;                                               // slots whose keys one of two streams has used
        struct Added { uint32_t low, high; } n0{0, 0}, n1{0, 0};           // halves of tiles whose values each stream has added
        int have = -1;                                                     // keys and values land in order: each is waited for once
        auto landed = [&](int item) {
            while (have < item) {
                ++have;
                if (!warp_wait(smem_u32(&kv_full[(uint32_t)have % S]), ((uint32_t)have / S) & 1, stop)) return false;
            }
            return true;
        };
        auto scores = [&](int u, int i) {
            const uint32_t slot = (2 * i) % S;
            const bool last = !PAIR || !(u ? st0 : st1).takes(i) || (scored >> slot & 1);
            mma_dot<DM>(lead, s_col + u * 128, q_desc + (PAIR ? u : 0) * (TILE >> 4), k_desc + slot * (TILE >> 4), IDESC_S);
            mma_commit(lead, smem_u32(&s_full[u]));
            if (last) mma_commit(lead, smem_u32(&kv_empty[slot]));
            scored = last ? scored & ~(1u << slot) : scored | 1u << slot;
        };
        auto weighted = [&](int u, int i, Added& n) {
            const Stream& st = u ? st1 : st0;
            const uint32_t slot = (2 * i + 1) % S;
            const int nx = st.next(i), key0 = kt.key(i, 128);
            // the weights are what is late: everything else is waited for first.  The next keys' slot was freed by products
            // that came before (a stream is at most two tiles ahead, and the ring holds five).
            if (!landed(nx <= st.upto ? 2 * nx : 2 * i + 1)) return false;
            if (st.sees_half(a, key0)) {
                if (!warp_wait(smem_u32(&p_full[u][0]), n.low & 1, stop)) return false;
                fence_after();
                mma_weighted<64>(lead, o_col + u * DM, p_col + u * p_step, v_desc + slot * (TILE >> 4), IDESC_O, n.low + n.high != 0);
                ++n.low;
            }
            if (st.sees_half(a, key0 + 64)) {
                if (!warp_wait(smem_u32(&p_full[u][1]), n.high & 1, stop)) return false;
                fence_after();
                mma_weighted<64>(lead, o_col + u * DM, p_col + u * p_step + 32, v_desc + slot * (TILE >> 4) + 4 * 128, IDESC_O, n.low + n.high != 0);
                ++n.high;
            }
            if (!PAIR || u == 1 || !st1.takes(i)) mma_commit(lead, smem_u32(&kv_empty[slot]));
            if (nx > st.upto) mma_commit(lead, smem_u32(&o_full[u]));
            if (nx <= st.upto) scores(u, nx);
            return true;
        };
        auto begin = [&](int u) {
            const int i = (u ? st1 : st0).begin();
            if (i > (u ? st1 : st0).upto) return true;
            if (!warp_wait(smem_u32(&q_full[PAIR ? u : 0]), 0, stop) || !landed(2 * i)) return false;
            fence_after();
            scores(u, i);
            return true;
        };
        ok = begin(0) && begin(1);
        for (int i = 0; i < kt.count && ok; ++i) {
            if (st0.takes(i)) ok = weighted(0, i, n0);
            if (ok && st1.takes(i)) ok = weighted(1, i, n1);
        }
        if (!ok) {                                                         // products in flight end before tensor memory is freed
            mma_commit(lead, smem_u32(&drained));
            mbar_wait(smem_u32(&drained), 0, 1u << 14);
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 9) tmem_free(tmem, 512);
    if (tid == 0 && stop_flag) report_stop(maps.timeouts, a.status);
}

template <typename T, int DM, bool PAIR, bool PAGED>
int launch(const SeqArgs& a, const FwdMaps& maps, dim3 grid, cudaStream_t st) {
    const cudaError_t e = cudaFuncSetAttribute(umma_fwd_kernel<T, DM, PAIR, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFwdSmem<DM>);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    umma_fwd_kernel<T, DM, PAIR, PAGED><<<grid, kThreads, kFwdSmem<DM>, st>>>(a, maps);
    count_tensor_launch();
    CA_CHECK_LAUNCH("window forward kernel (tensor cores)");
    return CA_OK;
}

template <bool PAGED>
int launch_any(const SeqArgs& a, const FwdMaps& maps, int dtype, bool pair, dim3 grid, cudaStream_t st) {
    const bool wide = a.D > 64;
#define CA_FWD(T)                                                                                                             \
    return wide ? (pair ? launch<T, 128, true, PAGED>(a, maps, grid, st) : launch<T, 128, false, PAGED>(a, maps, grid, st))   \
                : (pair ? launch<T, 64, true, PAGED>(a, maps, grid, st) : launch<T, 64, false, PAGED>(a, maps, grid, st))
    if (dtype == CA_BF16) CA_FWD(__nv_bfloat16);
    CA_FWD(__half);
#undef CA_FWD
}

}  // namespace

int encode_swizzled_map(CUtensorMap* map, bool bf16, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes,
                        const uint32_t* box) {
    typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<EncodeFn> cache{nullptr};
    EncodeFn fn = cache.load(std::memory_order_relaxed);
    if (!fn) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q);
        if (e != cudaSuccess || !sym) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return CA_ERR_CUDA; }
        fn = reinterpret_cast<EncodeFn>(sym);
        cache.store(fn, std::memory_order_relaxed);
    }
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    auto encode = [&] { return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                          dims, strides_bytes, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE); };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {           // a host thread whose first CUDA call this is: the runtime binds the device's context
        int dev = 0;
        if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
    }
    if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed with CUresult %d", (int)r); return CA_ERR_CUDA; }
    return CA_OK;
}

int encode_tokens(CUtensorMap* m, bool bf16, const ca_seq_view& v, int D, int heads, int tokens, int batch) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)tokens, (uint64_t)heads, (uint64_t)batch};
    const uint64_t strides[3] = {(uint64_t)v.token * 2, (uint64_t)v.head * 2, (uint64_t)v.batch * 2};
    const uint32_t box[4] = {64, 128, 1, 1};
    return encode_swizzled_map(m, bf16, v.data, 4, dims, strides, box);
}

int encode_rows(CUtensorMap* m, bool bf16, const ca_seq_view& v, const SeqArgs& a) {
    const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)a.Hq, (uint64_t)a.N, (uint64_t)a.B};
    const uint64_t strides[3] = {(uint64_t)v.head * 2, (uint64_t)v.token * 2, (uint64_t)(a.pages.table ? 16 : v.batch * 2)};
    const uint32_t box[4] = {64, (uint32_t)a.G, (uint32_t)(128 / a.G), 1};
    return encode_swizzled_map(m, bf16, v.data, 4, dims, strides, box);
}

// Maps of q, y and what rounding took, where tiles of rows are boxes; a negative scale turns the signs of q on the way.
static int encode_row_maps(FwdMaps* maps, bool bf16, const SeqArgs& a) {
    maps->rows = rows_fit(a) && !(a.scale < 0.f);
    if (!maps->rows) return CA_OK;
    int rc = encode_rows(&maps->q, bf16, a.q, a);
    if (!rc) rc = encode_rows(&maps->y, bf16, a.y, a);
    if (!rc && a.rest.data) rc = encode_rows(&maps->rest, bf16, a.rest, a);
    return rc;
}

// Two row tiles a CTA share the key tiles; where that leaves SMs idle, one row tile and two streams over its keys.
int umma_window_fwd(const SeqArgs& a, int dtype, cudaStream_t st) {
    FwdMaps maps{};
    const bool bf16 = dtype == CA_BF16;
    int rc;
    if ((rc = encode_tokens(&maps.k, bf16, a.k, a.D, a.Hkv, a.N, a.B)) || (rc = encode_tokens(&maps.v, bf16, a.v, a.D, a.Hkv, a.N, a.B)) ||
        (rc = encode_row_maps(&maps, bf16, a)))
        return rc;
    if (!(maps.timeouts = stage_timeout_counter())) return cuda_fail(cudaGetLastError(), "cudaGetSymbolAddress(stage timeouts)");
    const int64_t rows = (int64_t)a.N * a.G;
    const bool pair = (rows + 255) / 256 * a.Hkv * a.B >= sm_count();
    return launch_any<false>(a, maps, dtype, pair, dim3((unsigned)((rows + (pair ? 255 : 127)) / (pair ? 256 : 128)), a.Hkv, a.B), st);
}

int umma_paged(const SeqArgs& a, int dtype, cudaStream_t st) {
    FwdMaps maps{};
    const bool bf16 = dtype == CA_BF16;
    int box = 16;
    while (box < 128 && a.pages.page % (2 * box) == 0) box *= 2;
    maps.box = box;
    const ca_page_view* pools[2] = {&a.kp, &a.vp};
    for (int i = 0; i < 2; ++i) {
        const ca_page_view& p = *pools[i];
        const uint64_t dims[4] = {(uint64_t)a.D, (uint64_t)a.pages.page, (uint64_t)a.Hkv, (uint64_t)(a.pages.pages > 0 ? a.pages.pages : 1)};
        const uint64_t strides[3] = {(uint64_t)p.token * 2, (uint64_t)p.head * 2, (uint64_t)p.page * 2};
        const uint32_t b[4] = {64, (uint32_t)box, 1, 1};
        const int rc = encode_swizzled_map(i ? &maps.v : &maps.k, bf16, p.data, 4, dims, strides, b);
        if (rc) return rc;
    }
    const int rc = encode_row_maps(&maps, bf16, a);
    if (rc) return rc;
    if (!(maps.timeouts = stage_timeout_counter())) return cuda_fail(cudaGetLastError(), "cudaGetSymbolAddress(stage timeouts)");
    const bool pair = paged_tiles(a.N, a.G, a.pages.sequences, 256) * a.Hkv >= sm_count() && (int64_t)a.N * a.G > 128LL * a.pages.sequences;
    const int64_t tiles = paged_tiles(a.N, a.G, a.pages.sequences, pair ? 256 : 128);
    return launch_any<true>(a, maps, dtype, pair, dim3((unsigned)tiles, a.Hkv, 1), st);
}

}  // namespace ca
