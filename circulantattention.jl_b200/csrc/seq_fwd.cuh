// Attention on token sequences, forward, on the tensor cores (tcgen05): dense tensors and a paged cache, 16-bit types.
//
// A CTA takes tiles of 128 query rows of one key head and walks the tiles of 128 keys that they see, with a running maximum
// and sum per row.  Scores of a tile come into tensor memory (128 lanes = rows, 128 columns = keys); the thread that owns the
// row reads them, turns them into weights, and writes those back over the scores as 16-bit pairs, from where the second
// product takes them as its A operand: the weights never see shared memory.
//
// Roles: two groups of four (with a cap: eight) warps do the softmax, one warp copies keys and values by TMA into a ring of tiles, one warp
// issues the products.  The two groups are two streams that share the tensor cores: while one turns its scores into weights,
// the products of the other run.  With PAIR the streams are two row tiles that share every key tile (half the copies); without,
// they take the even and the odd key tiles of one row tile and are joined at the end (few rows).
//
// The accumulator is rescaled only where a row's maximum grew by more than 2^8 since its reference: the weights stay below
// 2^8 (of small caps in bfloat16, which have a fixed reference, below 2^32), and the products and sums are held in Float32.  Weights are rounded to the tensors' type before their product, once more
// than the result itself: errors are 1.15 to 1.6 of those of a plain implementation that keeps them in Float32.
//
// Bound: the exponentials and the products, 2048 cycles each for a pair of 128 x 128 tiles at 128 features; a pair takes about
// 3300 in the steady state, since a row's chain (scores, maximum, exponentials, weights) leaves gaps that two streams do not
// fill.  Measured: 65536 tokens, window 4096, 16 query and 2 key heads 2.03 ms (1.05 PFLOP/s of visible pairs; a
// large matrix product has 1.62 in a burst and keeps up 1.37; 1.99 to 2.14 ms by box, at the power cap); 2 x 16384 tokens, window 1024, 16 and 4 heads 415 us.
//
// Other scores and masks (FORM) are compiled apart.  What they cost: 16384 tokens, window 1024, 16 and 4 heads, bfloat16: plain 180 us,
// one document 224 (the remainders' product), slopes 246, cap 259 (282 with scores beyond the cap), both 336.  Bound: issue slots and
// the chain of a tile; a capped score takes 13 instructions, a plain one 7.  Packed training (16384 tokens in 13 documents, capped)
// 290 us.
#pragma once
#include "seq_umma.cuh"

#include <limits.h>

namespace ca {

struct FwdMaps {
    CUtensorMap k, v, q, y, rest;
    int rows;           // q, y and rest move by tiles of rows (maps), else by threads
    int box;            // paged: keys of a box
    int ranked;         // dense: the largest tiles first
    int* timeouts;
};

namespace {

// Warpgroups of softmax, a warp that copies and one that issues the products.  A stream has one warpgroup, a thread for each row; with
// a cap two, a thread for each row and half of the keys: that arithmetic is twice as much, and two warps on a scheduler leave
// half of its slots empty (16384 tokens, window 1024, bfloat16: cap 259 us with two, 284 with one, 297 and 359 where some scores
// lie beyond the cap; cap and slopes 341 and 354; but slopes alone 267 and 247, other masks 241 and 224: a tile costs a warp its
// waits whatever it does in it).
template <int FORM> constexpr int kGroups = has_cap(FORM) ? 2 : 1;
template <int FORM> constexpr int kSoftmaxWarps = 8 * kGroups<FORM>;
template <int FORM> constexpr int kThreads = 32 * (kSoftmaxWarps<FORM> + 2);

// Of capped scores that are read once: the same for all rows, 2^32 below the largest weight that the cap allows.  With cap_out up to
// kOnePassCap the smallest is 2^-64, so that neither the weights nor what they multiply leave Float32's exponents: a row's weighted
// sum is exact (but for the roundings) from 2^-62 on, and up to 2^95 of it, whatever the scores are.  Results are read with
// subnormal numbers taken for zeros, which is what a lower reference or a larger cap would run into first (all scores of a row near
// -cap, a cap of 50 and 2^20 in place of 2^32: values below 0.3 came out as zeros).
constexpr float kOnePassCap = 48.f;                 // in units of log2(e): a cap of 33
__device__ __forceinline__ float cap_reference(const SeqArgs& a) { return a.form.cap_out - 32.f; }

template <int DM> constexpr uint32_t kTileBytes = 128 * DM * 2;
template <int DM> constexpr int kSlots = DM == 128 ? 5 : 8;
template <int DM> constexpr size_t kFwdSmem = (size_t)(2 + kSlots<DM>) * kTileBytes<DM> + 1024;

// Whole numbers in the order of the Float32 ones, and back.
__device__ __forceinline__ int order_of(float x) {
    const int b = __float_as_int(x);
    return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float number_of(int o) { return __int_as_float(o ^ ((o >> 31) & 0x7fffffff)); }

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

template <bool PAIR, int FORM>
__device__ __forceinline__ Stream stream_of(const SeqArgs& a, const Seq& s, const KeyTiles& kt, int u, int r, int rows) {
    Stream t;
    t.lo = max(0, s.base + r / a.G);
    t.hi = r < rows ? min(s.n - 1, s.base + (min(r + 128, rows) - 1) / a.G) : -1;
    t.begin_key = max(0, tile_reach<FORM>(a, s, t.lo).lo);
    t.end_key = min(key_limit(a, s) - 1, t.hi < 0 ? -1 : tile_reach<FORM>(a, s, t.hi).hi);
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
    if (FORM) t.upto = min(t.upto, kt.count - 1);
    t.first = max(kt.first, min(min(t.from, t.upto + 1), firsts));
    return t;
}

template <typename T, int DM, bool PAIR, bool PAGED, int FORM>
__global__ void __launch_bounds__(kThreads<FORM>, 1) umma_fwd_kernel(const __grid_constant__ SeqArgs a, const __grid_constant__ FwdMaps maps) {
    // Dense calls with other scores or masks keep what rounding takes from the weights as a second 16-bit number, for one more
    // product with the values: where a few keys have most of the weight, their rounding would come out multiplied in delta = dy.y,
    // which the backward subtracts from each dy.v.  Calls over a cache have no gradients; there (ROUNDED) the weighted sum is divided
    // by the sum of the weights as they were rounded, so that the error of such weights nearly cancels.  Capped scores of standard
    // deviation 8, bfloat16: gradients off by 2.4e-3 of the norm with the second product, 2.6e-3 with the other sum, 3.5e-3 with
    // neither.
    constexpr bool SPLIT = FORM && !PAGED, ROUNDED = FORM && PAGED;
    // Capped weights are added 32 keys at a time, so that the products begin with the first while the others are made (packed training
    // 283 -> 272 us).
    constexpr bool QUARTERS = SPLIT && FORM == kCap;
    constexpr int GROUPS = kGroups<FORM>, WARPS = kSoftmaxWarps<FORM>, STREAM = 128 * GROUPS;      // STREAM: threads of a stream's softmax
    constexpr int S = kSlots<DM>;
    constexpr uint32_t TILE = kTileBytes<DM>;
    constexpr uint32_t IDESC_S = instr_desc(kIsBf16<T>, 128, false), IDESC_O = instr_desc(kIsBf16<T>, DM, true);
    extern __shared__ char raw[];
    __shared__ uint64_t kv_full[S], kv_empty[S], q_full[2], s_full[2], p_full[2][2], p_more[2][2], o_full[2], max_full[2], drained;
    __shared__ uint32_t tmem_slot, valid[S];
    __shared__ int stop_flag;
    __shared__ float merge_m[GROUPS == 1 ? 128 : 1], merge_l[GROUPS == 1 ? 128 : 1], merge_r[GROUPS == 1 && ROUNDED ? 128 : 1];
    __shared__ int row_max[GROUPS == 2 && FORM != kCap ? 2 : 1][128];      // ordered as the numbers (order_of)
    volatile int* stop = &stop_flag;

    const uint32_t raw_at = smem_u32(raw), base_at = (raw_at + 1023) & ~1023u;
    char* const smem = raw + (base_at - raw_at);
    const uint32_t q_at = base_at, kv_at = base_at + 2 * TILE;

    if (FORM && !PAGED) wait_for_previous();            // spans are made by the kernel before, which lets this one begin
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int tile = (int)(gridDim.x - 1 - blockIdx.x), h = blockIdx.y;       // the last rows see the most keys: first
    int2 owned;
    Seq s;
    if (PAGED) {
        owned = owned_tokens(a);
        if (!paged_seq(a, PAIR ? 256 : 128, tile, &s)) {
            if (tid < 32 * WARPS) clear_unowned<T>(a, owned, h, tid, 32 * WARPS);
            return;
        }
    } else {
        __shared__ int ranked;
        const bool rank = FORM && maps.ranked;
        const Place place = rank ? place_by_rank() : Place{tile, (int)blockIdx.y, (int)blockIdx.z};
        tile = place.x;
        h = place.h;
        s = dense_seq(a, place.b);
        if (rank)
            tile = ranked_tile(gridDim.x, tile, reinterpret_cast<int*>(smem + 2 * TILE), &ranked, [&](int first, int last) {
                return row_work<FORM>(a, s, first * (PAIR ? 256 : 128), (last + 1) * (PAIR ? 256 : 128));
            });
    }
    const int rows = s.T * a.G, R0 = tile * (PAIR ? 256 : 128);
    const int p_lo = max(0, s.base + R0 / a.G), p_hi = min(s.n - 1, s.base + (min(R0 + (PAIR ? 256 : 128), rows) - 1) / a.G);
    const KeyTiles kt = key_tiles<FORM>(a, s, p_lo, p_hi, 128);

    // Which key tiles a stream takes: with PAIR both see nearly the same, but each leaves out what all of its rows are blind to.
    const Stream st0 = stream_of<PAIR, FORM>(a, s, kt, 0, R0, rows), st1 = stream_of<PAIR, FORM>(a, s, kt, 1, PAIR ? R0 + 128 : R0, rows);

    if (warp == WARPS && lane == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        for (int u = 0; u < 2; ++u) {
            mbar_init(&q_full[u], maps.rows ? 1 : PAIR ? STREAM / 32 : WARPS);
            mbar_init(&s_full[u], 1);
            mbar_init(&p_full[u][0], GROUPS == 2 && FORM != kCap ? 8 : 4);        // the other half's threads rescale their columns of the sum
            mbar_init(&p_full[u][1], GROUPS == 2 && FORM != kCap ? 8 : 4);
            mbar_init(&p_more[u][0], 4);
            mbar_init(&p_more[u][1], 4);
            mbar_init(&o_full[u], 1);
            mbar_init(&max_full[u], STREAM / 32);
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
    if (GROUPS == 2 && FORM != kCap && tid < 256) row_max[tid >> 7][tid & 127] = order_of(-INFINITY);
    if (warp == WARPS + 1) tmem_alloc(smem_u32(&tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    // Scores of both streams, then their accumulators.  At 64 features there is room for weights beside the scores; at 128 they
    // overlay them, which needs the next scores to be written after the product with the weights has read them: products of
    // one shape (both 128 x 128 x 16 there) are carried out in the order of their issue.
    // Weights that are written by two warpgroups lie in the columns of their own scores: those of half a tile in its half.  With
    // remainders those of 32 keys lie in 16 columns and their remainders in the next 16.
    const uint32_t s_col = tmem, o_col = tmem + 256, p_col = DM == 64 ? tmem + 384 : s_col, p_step = DM == 64 ? 64 : 128, p_half = DM == 128 && (GROUPS == 2 || SPLIT) ? 64 : 32;
    static_assert(!SPLIT || DM == 128, "tensor memory has room for the remainders where weights lie over the scores");

    if (warp < WARPS) {
        // ------------------------------------------------------------ softmax: thread = row
        const int u = warp / (4 * GROUPS), g = GROUPS == 2 ? warp >> 2 & 1 : 0, r = tid & 127;      // stream, half of the keys, row
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
            constexpr int THREADS = PAIR ? STREAM : 2 * STREAM;
            const int t = tid % THREADS;
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
        // A capped score is at most cap log2(e): with a reference that all rows share (cap_reference) one pass over the scores is
        // enough.  Scores with a slope need the maximum of the changed ones, and
        // return to tensor memory in units of log2(e) for the exponentials (247 us; computed twice 288).
        constexpr bool BOUNDED = FORM == kCap, KEPT = has_slopes(FORM);
        const float sl2 = has_cap(FORM) || has_slopes(FORM) ? 1.f : a.mag_log2, cap_in = fabsf(a.form.cap_in);
        const float slope = has_slopes(FORM) ? slope_of(a, h * a.G + R - token_of(a, R) * a.G) : 0.f;
        const CapPoly<T> poly(a, cap_in, a.form.cap_out);
        const Reach mine = reach<FORM>(a, s, pos);
        const int doc_lo = document_of<FORM>(a, s, st.hi);
        const int c_lo = tile_reach<FORM>(a, s, p_lo).lo, c_hi = min(tile_reach<FORM>(a, s, p_hi).hi, s.n - 1);   // keys that any row of the CTA sees (or < sinks)
        // tiles from in_lo (or below in_sink) to in_hi need no mask
        const bool whole = st.lo == s.base + (R - r) / a.G && st.hi == s.base + (min(R - r + 128, rows) - 1) / a.G;
        const int in_hi = whole ? min(reach<FORM>(a, s, st.lo).hi, s.n - 1) - 127 : INT_MIN, in_lo = reach<FORM>(a, s, st.hi).lo, in_sink = a.sinks - 127;
        float m = -INFINITY, l = 0.f, lr = 0.f;            // ROUNDED: lr is the sum of the rounded weights
        int done = 0;
        bool ok = true;
        if (PAGED) clear_unowned<T>(a, owned, h, tid, 32 * WARPS);
        for (int i = st.begin(); i <= st.upto; i = st.next(i)) {
            const int key0 = kt.key(i, 128), vslot = (2 * i + 1) % S;
            const bool pads = FORM && (key0 < doc_lo || key0 + 127 > st.hi) && mixed<FORM>(a, s, key0, key0 + 127);
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
            const int hi = live ? min(mine.hi, s.n - 1) - key0 : -1, lo = mine.lo - key0, sk = a.sinks - key0;
            // Bits of the columns at .. at + 31 that the row sees
            auto seen = [&](int at) {
                uint32_t mk = seen_bits(lo - at, hi - at, sk - at);
                if (PAGED) mk &= ((there >> (at / 16)) & 1 ? 0xffffu : 0u) | ((there >> (at / 16 + 1)) & 1 ? 0xffff0000u : 0u);
                return mk;
            };
            // values that no row sees may be anything (a page that was freed, tokens behind the length, padding): zeros; of two
            // warpgroups each clears those of its half of the keys, which are all that the product with its weights reads
            if (!((key0 >= c_lo || far < a.sinks) && far <= c_hi && there == 0xff) || pads) {
                if (!PAGED && !warp_wait(smem_u32(&kv_full[vslot]), vpar, stop)) { ok = false; break; }
                const int j = key0 + r;
                if ((GROUPS == 1 || r >> 6 == g) && (!(j <= c_hi && (j >= c_lo || j < a.sinks) && (there >> (r >> 4) & 1)) || (pads && padding<FORM>(a, s, j)))) {
#pragma unroll 1
                    for (int p = 0; p < DM / 64; ++p)
#pragma unroll
                        for (int c = 0; c < 8; ++c)
                            *reinterpret_cast<uint4*>(smem + (2 + vslot) * TILE + p * kPanel + r * 128 + ((c ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            // Columns from..to - 1 of the weighted sum, by the factor of a new reference.  The scores came after the previous weighted
            // sum, which is therefore complete.
            auto rescale = [&](int from, int to, float f) {
#pragma unroll 1
                for (int c = from; c < to; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(O_at + c, o);
                    tmem_wait_ld();
                    settled32(o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st32(O_at + c, o);
                }
            };
            auto given = [&](float mx) {                                   // a reference for scores up to mx; the factor for what is there
                float f = 1.f;
                if (mx > m + 8.f) {                                        // also from -inf
                    f = fast_exp2(m - mx);
                    m = mx;
                }
                return f;
            };
            // What rounding took from a pair of weights, or the sum of the rounded ones
            auto remainder = [&](uint32_t w, float e0, float e1, f32x2& round2, uint32_t& rest) {
                float w0, w1;
                unpack16<T>(w, w0, w1);
                if (ROUNDED) round2 = add2(round2, pack2(w0, w1));
                if (SPLIT) {
                    unpack2(fma2(pack2(w0, w1), pack2(-1.f, -1.f), pack2(e0, e1)), w0, w1);
                    rest = pack16<T>(w0, w1);
                }
            };
            const int side = far <= st.lo ? 1 : key0 >= st.hi ? -1 : 0;    // of the keys, for all rows
            if constexpr (GROUPS == 1) {
                auto scores = [&](int g, uint32_t* x) {                    // the columns 64 g .. 64 g + 63
                    tmem_ld32(S_at + 64 * g, x);
                    tmem_ld32(S_at + 64 * g + 32, x + 32);
                    tmem_wait_ld();
                    settled32(x);
                    settled32(x + 32);
                };
                // The same for the maximum: -inf where the row does not see the key, written back for the exponentials
                auto masked_scores = [&](int g, uint32_t* x) {
                    scores(g, x);
                    if (has_slopes(FORM)) {
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            slope_scores<32>(x + 32 * q, a.mag_log2, slope, (float)(pos - key0 - 64 * g - 32 * q), side);
                    }
                    if (edge || KEPT) {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int at = 64 * g + 32 * q;
                            if (!KEPT || edge) {
                                const uint32_t mk = seen(at);
#pragma unroll
                                for (int c = 0; c < 32; ++c) x[32 * q + c] = (mk >> c) & 1 ? x[32 * q + c] : 0xff800000u;
                            }
                            tmem_st32(S_at + at, x + 32 * q);
                        }
                    }
                };
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
                const float before = m, f = given(mx * sl2);
                if (done && __any_sync(~0u, m != before)) rescale(0, DM, f);
                const float ref = m == -INFINITY ? 0.f : m;                // a row that has seen nothing yet
                const f32x2 sc2 = pack2(sl2, sl2), ref2 = pack2(-ref, -ref);
                f32x2 sum2 = pack2(l * f, 0.f), round2 = pack2(lr * f, 0.f);
#pragma unroll 1
                for (int g = 0; g < 2; ++g) {
                    if (!st.sees_half(a, key0 + 64 * g)) continue;
                    uint32_t x[64], w[32], rest[SPLIT ? 32 : 1];
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
                        if (ROUNDED || SPLIT) remainder(w[c], e0, e1, round2, rest[SPLIT ? c : 0]);
                    }
                    if (SPLIT) {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            tmem_st16(P_at + p_half * g + 32 * q, w + 16 * q);
                            tmem_st16(P_at + p_half * g + 32 * q + 16, rest + (SPLIT ? 16 * q : 0));
                        }
                    } else {
                        tmem_st32(P_at + p_half * g, w);
                    }                                                      // at 128 features over scores that this warp has read twice
                    tmem_wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&p_full[u][g]));   // the product with the first half may start
                }
                float a0, a1;
                unpack2(sum2, a0, a1);
                l = a0 + a1;
                unpack2(round2, a0, a1);
                lr = a0 + a1;
            } else {
                const bool own = st.sees_half(a, key0 + 64 * g), others = st.sees_half(a, key0 + 64 - 64 * g);
                // 32 columns from 64 g + 32 q as they go into the exponential, but for the reference; hidden ones are -inf
                auto scores = [&](int q, uint32_t* x, bool kept) {
                    const int at = 64 * g + 32 * q;
                    tmem_ld32(S_at + at, x);
                    tmem_wait_ld();
                    settled32(x);
                    if (kept) return;
                    const uint32_t mk = edge ? seen(at) : ~0u;
                    if (edge) clear_unseen<32>(x, mk);
                    if constexpr (BOUNDED)
                        poly.template scores<32>(x, -cap_reference(a), [&] {
                            tmem_ld32(S_at + at, x);
                            tmem_wait_ld();
                            settled32(x);
                        });
                    else cap_scores<T, 32>(x, cap_in, a.form.cap_out);
                    if (has_slopes(FORM)) slope_scores<32>(x, 1.f, slope, (float)(pos - key0 - at), side);
                    if (edge) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) x[c] = (mk >> c) & 1 ? x[c] : 0xff800000u;
                    }
                };
                float f = 1.f;
                if (BOUNDED) {
                    m = cap_reference(a);
                } else {
                    float mx = -INFINITY;
                    if (own) {
#pragma unroll 1
                        for (int q = 0; q < 2; ++q) {
                            uint32_t x[32];
                            scores(q, x, false);
                            tmem_st32(S_at + 64 * g + 32 * q, x);
                            float top[2] = {mx, -INFINITY};
#pragma unroll
                            for (int c = 0; c < 32; c += 4)
#pragma unroll
                                for (int e = 0; e < 2; ++e) top[e] = fmaxf(fmaxf(top[e], __uint_as_float(x[c + e])), __uint_as_float(x[c + 2 + e]));
                            mx = fmaxf(top[0], top[1]);
                        }
                    }
                    tmem_wait_st();
                    // The largest of all tiles so far, of both halves: a number for each row is all that fits beside the tiles
                    atomicMax(&row_max[u][r], order_of(mx));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&max_full[u]));
                    if (!warp_wait(smem_u32(&max_full[u]), done & 1, stop)) { ok = false; break; }
                    const float before = m;
                    f = given(number_of(*(volatile int*)&row_max[u][r]));
                    if (done && __any_sync(~0u, m != before)) rescale(DM / 2 * g, DM / 2 * (g + 1), f);
                    tmem_wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0 && others) mbar_arrive(smem_u32(&p_full[u][1 - g]));
                }
                if (own) {
                    const float ref = m == -INFINITY ? 0.f : m;            // a row that has seen nothing yet
                    const f32x2 ref2 = pack2(-ref, -ref);
                    f32x2 sum2 = pack2(l * f, 0.f), round2 = pack2(lr * f, 0.f);
#pragma unroll 1
                    for (int q = 0; q < 2; ++q) {
                        uint32_t x[32], w[16], rest[SPLIT ? 16 : 1];
                        scores(q, x, KEPT);
#pragma unroll
                        for (int c = 0; c < 16; ++c) {
                            float e0, e1;
                            if (BOUNDED) e0 = __uint_as_float(x[2 * c]), e1 = __uint_as_float(x[2 * c + 1]);
                            else unpack2(add2(pack2(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1])), ref2), e0, e1);
                            e0 = fast_exp2(e0);             // the cap's polynomial fills the FMA pipe: none of these on it
                            e1 = fast_exp2(e1);
                            sum2 = add2(sum2, pack2(e0, e1));
                            w[c] = pack16<T>(e0, e1);
                            remainder(w[c], e0, e1, round2, rest[SPLIT ? c : 0]);
                        }
                        const uint32_t to = P_at + p_half * g + (SPLIT ? 32 : 16) * q;
                        tmem_st16(to, w);
                        if (SPLIT) tmem_st16(to + 16, rest);
                        if (QUARTERS || q) {
                            tmem_wait_st();
                            fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(QUARTERS && q ? &p_more[u][g] : &p_full[u][g]));
                        }
                    }
                    float a0, a1;
                    unpack2(sum2, a0, a1);
                    l = a0 + a1;
                    unpack2(round2, a0, a1);
                    lr = a0 + a1;
                } else {
                    l *= f;
                    lr *= f;
                }
            }
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
        if (!PAIR || keep_rest || GROUPS == 2) group_sync<2 * STREAM>(1);  // both streams are through with the ring
        // two warpgroups: what their halves of the keys summed up, in the ring's last slot; the reference is the same
        float* const sums = reinterpret_cast<float*>(smem + (1 + S) * TILE);                // [stream][half][row]
        if (GROUPS == 2) {
            sums[(2 * u + g) * 128 + r] = l;
            sums[512 + (2 * u + g) * 128 + r] = lr;
            sums[1024 + u * 128 + r] = m;
            group_sync<2 * STREAM>(1);
            l = sums[2 * u * 128 + r] + sums[(2 * u + 1) * 128 + r];
            lr = sums[512 + 2 * u * 128 + r] + sums[512 + (2 * u + 1) * 128 + r];
        }
        const int col_from = DM / GROUPS * g, col_to = DM / GROUPS * (g + 1);               // the thread's columns of the results
        if (!PAIR) {
            if (u == 1) {
                if (GROUPS == 1) {
                    merge_m[r] = m;
                    merge_l[r] = l;
                    if (ROUNDED) merge_r[r] = lr;
                }
                if (done && ok) {
#pragma unroll 1
                    for (int c = col_from; c < col_to; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(O_at + c, o);
                        tmem_wait_ld();
                        settled32(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) other[(c + e) * 128 + r] = __uint_as_float(o[e]);
                    }
                }
            }
            group_sync<2 * STREAM>(1);
            const float m1 = GROUPS == 2 ? sums[1024 + 128 + r] : merge_m[r], l1 = GROUPS == 2 ? sums[256 + r] + sums[384 + r] : merge_l[r];
            const float M = fmaxf(m, m1), ref = M == -INFINITY ? 0.f : M;
            f0 = fast_exp2(m - ref);
            f1 = fast_exp2(m1 - ref);
            l = l * f0 + l1 * f1;
            if (ROUNDED) lr = lr * f0 + (GROUPS == 2 ? sums[512 + 256 + r] + sums[512 + 384 + r] : merge_r[r]) * f1;
            m = M;
        }
        if (PAIR || u == 0) {
            const float total = ROUNDED ? lr : l;
            float inv = total > 0.f ? 1.f / total : 0.f;
            if (!ok || *stop) inv = __int_as_float(0x7fffffff);            // a wait ran out: NaN, never a wrong number
            // Rows that see nothing are zeros by choice, not by their weights: 0 * inf of a value that other rows see is not a number.
            const bool none = !done || l == 0.f, both = !PAIR && kt.count > 1 && !none;
            if (!PAGED && a.lse && have && g == 0) a.lse[((int64_t)s.b * a.Hkv + h) * rows + R] = l > 0.f ? m + log2f(l) : -INFINITY;
            const float w0 = f0 * inv, w1 = f1 * inv;
            // y goes to the queries' place (their last scores are done), what rounding took to a slot of the ring
            const int tile0 = R - r;
            char *const out = smem + (PAIR ? u : 0) * TILE, *const out_rest = smem + (2 + (PAIR ? u : 2)) * TILE;
#pragma unroll 1
            for (int c = col_from; c < col_to; c += 32) {
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
            group_sync<STREAM>(2 + u);
            // by maps, which leave out tokens behind the tensor's; a cache's packed rows go on with the next sequence
            if (maps.rows && (!PAGED || tile0 + 128 <= rows)) {
                if (r == 0 && g == 0 && tile0 < rows) {
                    const int token = s.t0 + tile0 / a.G, b = PAGED ? 0 : s.b;
#pragma unroll
                    for (int p = 0; p < DM / 64; ++p) {
                        if (FORM && 64 * p >= a.D) break;                  // few features in a kernel for 128
                        tma_store_4d(&maps.y, smem_u32(out) + p * kPanel, 64 * p, h * a.G, token, b);
                        if (keep_rest) tma_store_4d(&maps.rest, smem_u32(out_rest) + p * kPanel, 64 * p, h * a.G, token, b);
                    }
                    tma_stores_read();
                }
            } else {
                auto row = [&](const ca_seq_view& v) { return [&](int rr) { return seq_row<T>(v, a, s, h, max(tile0 + rr, 0)); }; };
                store_tile<T, DM, STREAM>(out, row(a.y), rows - tile0, a.D, tid % STREAM);
                if (keep_rest) store_tile<T, DM, STREAM>(out_rest, row(a.rest), rows - tile0, a.D, tid % STREAM);
            }
        }
    } else if (warp == WARPS) {
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
    } else if (warp == WARPS + 1) {
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
            const bool low = st.sees_half(a, key0), high = st.sees_half(a, key0 + 64);
            const uint32_t to = o_col + u * DM, from = p_col + u * p_step;
            const uint64_t values = v_desc + slot * (TILE >> 4);
            bool add = n.low + n.high != 0;
            // the weights of 32 keys and their remainders, quarter q of the tile
            auto add_quarter = [&](uint32_t q) {
                mma_weighted<32>(lead, to, from + 32 * q, values + q * (2 * 128), IDESC_O, add);
                mma_weighted<32>(lead, to, from + 32 * q + 16, values + q * (2 * 128), IDESC_O, true);
                add = true;
            };
            auto add_half = [&](uint32_t half) {
                if (!warp_wait(smem_u32(&p_full[u][half]), (half ? n.high : n.low) & 1, stop)) return false;
                fence_after();
                if (SPLIT) {
                    add_quarter(2 * half);
                    add_quarter(2 * half + 1);
                } else {
                    mma_weighted<64>(lead, to, from + p_half * half, values + half * (4 * 128), IDESC_O, add);
                    add = true;
                }
                return true;
            };
            if (QUARTERS) {
#pragma unroll
                for (uint32_t q = 0; q < 2; ++q)                           // the two halves are made at the same time
#pragma unroll
                    for (uint32_t half = 0; half < 2; ++half) {
                        if (!(half ? high : low)) continue;
                        if (!warp_wait(smem_u32(q ? &p_more[u][half] : &p_full[u][half]), (half ? n.high : n.low) & 1, stop)) return false;
                        fence_after();
                        add_quarter(2 * half + q);
                    }
            } else {
                if (low && !add_half(0)) return false;
                if (high && !add_half(1)) return false;
            }
            n.low += low;
            n.high += high;
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
        // The second stream's rows may be of a document that begins many tiles behind the first stream's: its first keys are
        // waited for one tile ahead, when the ring has come to them.
        bool late = FORM && PAIR && st1.begin() > 1;
        ok = begin(0) && (late || begin(1));
        for (int i = 0; i < kt.count && ok; ++i) {
            if (late && st1.begin() <= i + 1) {
                late = false;
                if (!(ok = begin(1))) break;
            }
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
    if (warp == WARPS + 1) tmem_free(tmem, 512);
    if (tid == 0 && stop_flag) report_stop(maps.timeouts, a.status);
}

template <typename T, int DM, bool PAIR, bool PAGED, int FORM>
int launch(const SeqArgs& a, const FwdMaps& maps, dim3 grid, cudaStream_t st) {
    const cudaError_t e = cudaFuncSetAttribute(umma_fwd_kernel<T, DM, PAIR, PAGED, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFwdSmem<DM>);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    if (FORM && !PAGED) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid; cfg.blockDim = dim3(kThreads<FORM>); cfg.dynamicSmemBytes = kFwdSmem<DM>; cfg.stream = st;
        cfg.attrs = at; cfg.numAttrs = 1;
        const cudaError_t l = cudaLaunchKernelEx(&cfg, umma_fwd_kernel<T, DM, PAIR, PAGED, FORM>, a, maps);
        if (l != cudaSuccess) return cuda_fail(l, "window forward kernel (tensor cores)");
    } else {
        umma_fwd_kernel<T, DM, PAIR, PAGED, FORM><<<grid, kThreads<FORM>, kFwdSmem<DM>, st>>>(a, maps);
    }
    count_tensor_launch();
    CA_CHECK_LAUNCH("window forward kernel (tensor cores)");
    return CA_OK;
}

template <bool PAGED, int FORM>
int launch_any(const SeqArgs& a, const FwdMaps& maps, int dtype, bool pair, dim3 grid, cudaStream_t st) {
    const bool wide = a.D > 64 || (FORM && !PAGED);
#define CA_FWD(T)                                                                                                              \
    if (wide) return pair ? launch<T, 128, true, PAGED, FORM>(a, maps, grid, st) : launch<T, 128, false, PAGED, FORM>(a, maps, grid, st); \
    if constexpr (!FORM || PAGED) return pair ? launch<T, 64, true, PAGED, FORM>(a, maps, grid, st) : launch<T, 64, false, PAGED, FORM>(a, maps, grid, st)
    if (dtype == CA_BF16) { CA_FWD(__nv_bfloat16); }
    if constexpr (FORM != kCap) { CA_FWD(__half); }                        // half takes kCapSlopes (seq_fwd.cu)
    return CA_ERR_UNSUPPORTED;
#undef CA_FWD
}

}  // namespace

// All variants of one kind.
template <int FORM>
int umma_fwd(const SeqArgs& a, const FwdMaps& maps, int dtype, bool pair, dim3 grid, cudaStream_t st) {
    return a.pages.table ? launch_any<true, FORM>(a, maps, dtype, pair, grid, st) : launch_any<false, FORM>(a, maps, dtype, pair, grid, st);
}

}  // namespace ca
