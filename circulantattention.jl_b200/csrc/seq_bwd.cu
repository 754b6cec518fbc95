// Attention on token sequences, backward, on the tensor cores (tcgen05), 16-bit types, no atomics.
//
// With P = 2^(scale log2(e) q.k - lse), dP = dy.v and delta = dy.y:  dS = P (dP - delta),
//     dq = scale dS k,   dk = scale dS^T q,   dv = P^T dy.
// dq needs the sum over keys, dk and dv the sum over queries.  One sweep that did both would add one of the two into
// memory from many CTAs, in an order that changes; two sweeps recompute two of seven products instead and stay exact in
// their order: the first owns 128 query rows, the second 128 keys.
//
// In both, four warpgroups share each 128 x 128 tile: a thread owns one lane (row / key) and 32 of the columns.  The
// weights return to tensor memory as 16-bit pairs and are the A operand of the next product from there.
//
// Bound: the products at 128 features, 1536 cycles a tile (dq) and 2048 (dk, dv); measured 2100 and 2800, the rest is the
// chain scores - weights - dS - product of one tile, of which neither tensor memory (all 512 columns are taken) nor shared memory
// holds a second.  Short windows are bound by what stands before the first tile (queries, results and their remainders
// from memory: 9000 cycles).  2 x 16384 tokens, window 1024, 16 query and 4 key heads: 502 and 543 us; 3 x 5001 tokens, 8 heads of
// 64 features, window 127, half: 59 and 60 us.
//
// With a cap dS has its derivative too: dS = P (dP - delta) (1 - tanh^2); a bias by distance changes P alone.  A weight then takes
// five packed products more (polynomial and derivative), and a look for scores beyond the cap: 16384 tokens, window 1024, 16 and 4
// heads, bfloat16: 252 and 280 us without, 317 and 362 with a cap, 267 and 303 with slopes.  Packed training (13 documents, capped):
// dq 324, dk and dv 322 us, of 20 and 20 instructions a score; a third of dq's stand before its first tile.
#include "seq_umma.cuh"

#include <limits.h>

namespace ca {
namespace {

// Four warpgroups that compute, each for a quarter of a tile's columns, and warps that copy, issue products and fetch the rows'
// sums.
constexpr int kGroups = 4, kCols = 128 / kGroups, kWork = 128 * kGroups, kWarps = 4 * kGroups, kThreads = kWork + 96;
constexpr int kCopier = kWarps, kIssuer = kWarps + 1, kFetcher = kWarps + 2;
template <int DM> constexpr uint32_t kTileBytes = 128 * DM * 2;
template <int DM> constexpr int kSlots = DM == 128 ? 5 : 8;
template <int DM> constexpr size_t kBwdSmem = (size_t)(2 + kSlots<DM>) * kTileBytes<DM> + 1024;

struct BwdMaps {
    CUtensorMap k, v, q, dy;
    CUtensorMap q_rows, dy_rows, y_rows, rest_rows, dq_rows, dk, dv;
    int sms;                // dq: the CTA so many further on takes this one's place
    int ranked;             // dk, dv: the largest tiles first
    int rows;               // q, dy and dq of the first sweep move by tiles of rows (maps), else by threads
    int* timeouts;
    float *dy_peak, *v_peak;    // half: largest magnitudes of each tile of 128 query rows / keys, [b][key head][tile]
    float* partial;         // [b][key head][tile][segment][dk, dv][feature][128 keys]
    int split_tiles;        // the first key tiles, whose queries are dealt to
    int segments;           // so many CTAs
};

// Half precision has too few exponents for the weights of long windows and for dS of scaled losses.  P is at most 1 and goes
// into its product as 2^8 P.  dS goes in as c dS with c = 2^(7 - floor(log2 max|dy|) - floor(log2 max|v|)): since
// P_j |v_j - sum P v| <= max|v| / 2, |dS| is at most 128 max|dy| max|v| / 2 for 128 features, and |c dS| < 2^15; and where dP
// is of the usual size, weights down to 2^-20 still give normal numbers.  max|v| is that of every key that the queries see, in
// dk too: through delta the values of all of them are in dS, whatever the size of the CTA's own.  Both factors are powers of two and
// leave with the results.  The peaks cost one pass over v (5 us for 32 MB).  bfloat16 has the exponents of Float32 and needs none
// of this.
constexpr float kPScale = 256.f, kPLog2 = 8.f;
__device__ __forceinline__ int exponent(float x) { return x > 0.f && !isinf(x) ? (int)(__float_as_uint(x) >> 23) - 127 : 0; }
__device__ __forceinline__ float ds_factor(float dy_peak, float v_peak) {
    return __uint_as_float((uint32_t)(127 + 7 - exponent(dy_peak) - exponent(v_peak)) << 23);      // halves: -24 <= exponents <= 15
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}

__device__ __forceinline__ void read_columns(uint32_t at, uint32_t* x) {
    tmem_ld32(at, x);
    tmem_wait_ld();
    settled32(x);
}

// 16 columns of either half of a tile's 128
__device__ __forceinline__ void read_halves(uint32_t at, uint32_t* x) {
    tmem_ld16(at, x);
    tmem_ld16(at + 64, x + 16);
    tmem_wait_ld();
    settled32(x);
}

template <int DM>
__device__ __forceinline__ void clear_row(char* tile, int r) {
#pragma unroll
    for (int p = 0; p < DM / 64; ++p)
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + p * kPanel + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
}

template <int FORM>
__global__ void __launch_bounds__(256) peak_kernel(const __grid_constant__ SeqArgs a, float* __restrict__ peaks) {
    __shared__ float part[8];
    const Seq s = dense_seq(a, blockIdx.z);
    const int pieces = a.D / 8, key0 = blockIdx.x * 128;
    const __half* v = (const __half*)a.v.data + blockIdx.y * a.v.head + s.b * a.v.batch;
    float peak = 0.f;
    for (int i = threadIdx.x; i < 128 * pieces; i += 256) {
        const int j = key0 + i / pieces;
        if (j >= s.n) break;
        if (padding<FORM>(a, s, j)) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(v + (int64_t)j * a.v.token + i % pieces * 8);
        const uint32_t* p = &w.x;
#pragma unroll
        for (int k = 0; k < 4; ++k) peak = fmaxf(peak, fmaxf(fabsf(low16<__half>(p[k])), fabsf(high16<__half>(p[k]))));
    }
    peak = warp_max(peak);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = peak;
    __syncthreads();
    if (threadIdx.x < 32) {
        peak = warp_max(threadIdx.x < 8 ? part[threadIdx.x] : 0.f);
        if (threadIdx.x == 0) peaks[((int64_t)s.b * a.Hkv + blockIdx.y) * gridDim.x + blockIdx.x] = peak;
    }
}

// ---------------------------------------------------------------- dq
// Tensor memory: scores 0..127, dP 128..255, dS 256..319, the queries 320..383, dq from 384.  While the warpgroups turn tile i
// into dS, the products of tile i + 1 run.
//
// The queries move into tensor memory, and their place becomes one more slot of the ring: a tile of keys stays until its product
// with dS, two steps behind its scores, so that with five slots the values of every tile came late (2450 cycles a tile; 1536
// are products).
template <typename T, int DM, int FORM>
__global__ void __launch_bounds__(kThreads, 1) umma_dq_kernel(const __grid_constant__ SeqArgs a, const __grid_constant__ BwdMaps maps) {
    constexpr int S = kSlots<DM> + 1;
    constexpr uint32_t TILE = kTileBytes<DM>;
    constexpr uint32_t IDESC_S = instr_desc(kIsBf16<T>, 128, false), IDESC_O = instr_desc(kIsBf16<T>, DM, true);
    extern __shared__ char raw[];
    __shared__ uint64_t kv_full[S], kv_empty[S], q_full, q_moved, s_full, s_free, dp_full, dp_free, ds_full, dq_done, o_full, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int stop_flag;
    __shared__ float part[2][128], warp_peak[4];
    volatile int* stop = &stop_flag;
    const uint32_t raw_at = smem_u32(raw), base_at = (raw_at + 1023) & ~1023u;
    char* const smem = raw + (base_at - raw_at);
    const uint32_t kv_at = base_at + TILE, q_at = kv_at + (S - 1) * TILE;    // dy, then the ring; the queries come into its last slot
    char* const q_tile = smem + S * TILE;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    const Seq s = dense_seq(a, blockIdx.z);
    const int rows = s.T * a.G, R0 = (int)(gridDim.x - 1 - blockIdx.x) * 128;
    const int f_lo = R0 / a.G, f_hi = (min(R0 + 128, rows) - 1) / a.G;      // tokens of the tile
    const int p_hi = min(s.n - 1, f_hi);
    const KeyTiles kt = key_tiles<FORM>(a, s, f_lo, f_hi, 128);

    if (warp == kCopier && lane == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&kv_full[i], 1); mbar_init(&kv_empty[i], 1); }
        mbar_init(&q_full, maps.rows ? 1 : kWarps);
        mbar_init(&q_moved, kWarps);
        mbar_init(&s_full, 1);
        mbar_init(&s_free, kWarps);
        mbar_init(&dp_full, 1);
        mbar_init(&dp_free, kWarps);
        mbar_init(&ds_full, kWarps);
        mbar_init(&dq_done, 1);
        mbar_init(&o_full, 1);
        mbar_init(&drained, 1);
        stop_flag = 0;
        mbar_fence_init();
        fence_async_smem();
        if (maps.rows) {                                       // on their way while the rest is set up
            mbar_arrive_expect_tx(smem_u32(&q_full), 2 * TILE);
#pragma unroll
            for (int p = 0; p < DM / 64; ++p) {
                tma_load_4d(q_at + p * kPanel, &maps.q_rows, 64 * p, h * a.G, R0 / a.G, s.b, smem_u32(&q_full));
                tma_load_4d(base_at + p * kPanel, &maps.dy_rows, 64 * p, h * a.G, R0 / a.G, s.b, smem_u32(&q_full));
            }
        }
        prefetch_map(&maps.k);
        prefetch_map(&maps.v);
    }
    if (warp == kIssuer) tmem_alloc(smem_u32(&tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot, q_col = tmem + 320, o_col = tmem + 384;

    if (warp < kWarps) {
        const int u = warp >> 2, r = tid & 127, R = R0 + r, pos = token_of(a, R);
        const bool have = R < rows, live = have && pos < s.n && !padding<FORM>(a, s, pos);
        const int64_t stat = ((int64_t)s.b * a.Hkv + h) * rows + R;
        const float lse = live ? a.lse[stat] : 0.f;
        const uint32_t lane_off = (uint32_t)(warp & 3) << 21;
        float delta, c = 1.f;
        {
            typedef TileCopy<DM, kWork> C;
            auto row = [&](const ca_seq_view& v) {
                return [&](int rr) { return seq_row<T>(v, a, s, h, min(R0 + rr, rows - 1)); };
            };
            const int to = (int)min((int64_t)rows, (int64_t)s.n * a.G) - R0;
            uint4 w[C::kCount], y[C::kCount], e[C::kCount];
            if (!maps.rows) {
                fetch_tile<T, DM, kWork>(y, row(a.q), 0, to, a.D, tid);
                fetch_tile<T, DM, kWork>(w, row(a.dy), 0, to, a.D, tid);
                put_tile<DM, kWork>(q_tile, y, tid);
                put_tile<DM, kWork>(smem, w, tid);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&q_full));
            }
            fetch_tile<T, DM, kWork>(y, row(a.y), 0, to, a.D, tid);
            if (a.rest.data) fetch_tile<T, DM, kWork>(e, row(a.rest), 0, to, a.D, tid);
            warp_wait(smem_u32(&q_full), 0, stop);                             // a wait that ran out shows at the next one
            if (32 * u < DM) {                                                 // features 32 u .. 32 u + 31 of the row
                uint32_t x[16];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<uint4*>(x + 4 * k) = *reinterpret_cast<const uint4*>(q_tile + C::at(r, 4 * u + k));
                tmem_st16(q_col + lane_off + 16 * u, x);
                tmem_wait_st();
                fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_moved));
            if (maps.rows) {
#pragma unroll
                for (int i = 0; i < C::kCount; ++i) {
                    w[i] = *reinterpret_cast<const uint4*>(smem + C::at(C::row(tid, i), C::piece(tid)));
                    if (C::row(tid, i) >= to) w[i] = make_uint4(0, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < C::kCount; ++i) {
                if (!a.rest.data) e[i] = make_uint4(0, 0, 0, 0);
                const uint32_t *pw = &w[i].x, *py = &y[i].x, *pe = &e[i].x;
                float d = 0.f, peak = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    d = fmaf(low16<T>(pw[k]), low16<T>(py[k]) + low16<T>(pe[k]), d);
                    d = fmaf(high16<T>(pw[k]), high16<T>(py[k]) + high16<T>(pe[k]), d);
                    if (!kIsBf16<T>) peak = fmaxf(peak, fmaxf(fabsf(low16<T>(pw[k])), fabsf(high16<T>(pw[k]))));
                }
#pragma unroll
                for (int o = C::kPieces / 2; o; o >>= 1) {
                    d += __shfl_xor_sync(~0u, d, o);
                    if (!kIsBf16<T>) peak = fmaxf(peak, __shfl_xor_sync(~0u, peak, o));
                }
                if (C::piece(tid) == 0) {
                    part[0][C::row(tid, i)] = d;
                    part[1][C::row(tid, i)] = peak;
                }
            }
            group_sync<kWork>(1);
            delta = !FORM || live ? part[0][r] : 0.f;
            if (u == 0 && have) a.delta[stat] = delta;
            if (!kIsBf16<T>) {
                float peak = !FORM || live ? part[1][r] : 0.f, v_peak = 0.f;
                const float* p = maps.v_peak + ((int64_t)s.b * a.Hkv + h) * ((a.N + 127) / 128);
                for (int i = lane; i < kt.count; i += 32) v_peak = fmaxf(v_peak, p[kt.key(i, 128) / 128]);
                c = ds_factor(peak, warp_max(v_peak));
                peak = warp_max(peak);
                if (u == 0 && lane == 0) warp_peak[warp] = peak;
            }
        }
        const float factor = has_cap(FORM) ? a.form.cap_out : a.scale_log2;
        const float sign = has_cap(FORM) ? -1.f : 1.f;             // with a cap x is P (tanh^2 - 1)
        const f32x2 sc2 = pack2(a.scale_log2, a.scale_log2), lse2 = pack2(-lse, -lse), dl2 = pack2(-delta * c * sign, -delta * c * sign), c2 = pack2(c * sign, c * sign);
        const float slope = has_slopes(FORM) ? slope_of(a, h * a.G + R - pos * a.G) : 0.f;
        const CapPoly<T> poly(a, a.form.cap_in, 1.f);
        const Reach mine = reach<FORM>(a, s, pos);
        const bool row_pads = mixed<FORM>(a, s, f_lo, f_hi);
        const int doc_lo = document_of<FORM>(a, s, p_hi);
        const int in_hi = reach<FORM>(a, s, f_lo).hi, in_lo = reach<FORM>(a, s, p_hi).lo;      // tiles from in_lo to in_hi need no mask
        const uint32_t S_at = tmem + kCols * u + lane_off, dp_at = S_at + 128, ds_at = tmem + 256 + kCols / 2 * u + lane_off;
        bool ok = true;
        for (int i = 0; i < kt.count; ++i) {
            const int key0 = kt.key(i, 128), far = key0 + 127;
            if (!warp_wait(smem_u32(&s_full), i & 1, stop)) { ok = false; break; }
            fence_after();
            uint32_t x[kCols];
            read_columns(S_at, x);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_free));
            uint32_t mk = ~0u;
            const bool pads = FORM && (key0 < doc_lo || far > p_hi) && mixed<FORM>(a, s, key0, far);
            const bool ragged = far >= s.n || f_hi != p_hi || pads || row_pads;      // the tile holds keys or rows that may be anything
            const bool edge = !(far <= in_hi && far < s.n && f_hi == p_hi && (key0 >= in_lo || far < a.sinks));
            if (edge) {
                const int hi = live ? min(mine.hi, s.n - 1) - key0 : -1, lo = mine.lo - key0, sk = a.sinks - key0;
                mk = seen_bits(lo - kCols * u, hi - kCols * u, sk - kCols * u);
            }
            if (has_cap(FORM) || has_slopes(FORM)) {
                f32x2 inner[has_cap(FORM) ? kCols / 2 : 1];    // P (1 - tanh^2) is all that dS needs
                if (has_cap(FORM) && edge) clear_unseen<kCols>(x, mk);
                if (FORM == kCap) poly.template scores<kCols>(x);
                else if (has_cap(FORM)) cap_scores<T, kCols>(x, a.form.cap_in, 1.f);
                if (has_cap(FORM)) cap_inner<kCols>(inner, x);
                if (has_slopes(FORM)) slope_scores<kCols>(x, factor, slope, (float)(pos - key0 - kCols * u), far <= f_lo ? 1 : key0 >= f_hi ? -1 : 0);
                const f32x2 f2 = has_slopes(FORM) ? pack2(1.f, 1.f) : pack2(factor, factor);
#pragma unroll
                for (int c = 0; c < kCols; c += 2) {
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), f2, lse2), e0, e1);
                    e0 = fast_exp2(e0);
                    e1 = fast_exp2(e1);
                    if (has_cap(FORM)) unpack2(mul2(pack2(e0, e1), inner[c / 2]), e0, e1);
                    x[c] = __float_as_uint(e0);
                    x[c + 1] = __float_as_uint(e1);
                }
            } else {
#pragma unroll
                for (int c = 0; c < kCols; c += 2) {
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sc2, lse2), e0, e1);
                    x[c] = __float_as_uint(fast_exp2(e0));
                    x[c + 1] = __float_as_uint(fast_exp2(e1));
                }
            }
            if (edge) {
                clear_unseen<kCols>(x, mk);
                if ((far >= s.n || pads) && u == 0) {          // keys behind the length, and padding, may be anything: zeros
                    const int slot = (2 * i) % S;              // the scores are there, so the keys are
                    if (key0 + r >= s.n || (pads && padding<FORM>(a, s, key0 + r))) clear_row<DM>(smem + (1 + slot) * TILE, r);
                    fence_async_smem();
                }
            }
            if (!warp_wait(smem_u32(&dp_full), i & 1, stop)) { ok = false; break; }
            fence_after();
            uint32_t y[kCols], w[kCols / 2];
            read_columns(dp_at, y);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&dp_free));
#pragma unroll
            for (int c = 0; c < kCols; c += 2) {
                float e0, e1;
                unpack2(mul2(fma2(pack2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), c2, dl2), pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1]))), e0, e1);
                y[c] = __float_as_uint(e0);
                y[c + 1] = __float_as_uint(e1);
            }
            if (ragged) clear_unseen<kCols>(y, mk);                   // dP of such pairs may be anything
#pragma unroll
            for (int c = 0; c < kCols; c += 2) w[c >> 1] = pack16<T>(__uint_as_float(y[c]), __uint_as_float(y[c + 1]));
            if (i && !warp_wait(smem_u32(&dq_done), (i - 1) & 1, stop)) { ok = false; break; }
            fence_after();
            tmem_st16(ds_at, w);
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ds_full));
        }
        if (kt.count && ok) ok = warp_wait(smem_u32(&o_full), 0, stop);
        fence_after();
        const float f = !ok || *stop ? __int_as_float(0x7fffffff) : a.scale / c;
        if (!kIsBf16<T>) {
            group_sync<kWork>(1);
            if (tid == 0)
                maps.dy_peak[((int64_t)s.b * a.Hkv + h) * gridDim.x + R0 / 128] = fmaxf(fmaxf(warp_peak[0], warp_peak[1]), fmaxf(warp_peak[2], warp_peak[3]));
        }
#pragma unroll 1
        for (int col = 32 * u; col < DM; col += 32 * kGroups) {
            uint32_t o[32];
            tmem_ld32(o_col + lane_off + col, o);
            tmem_wait_ld();
            settled32(o);
            float y[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = kt.count && live ? __uint_as_float(o[e]) * f : 0.f * f;      // behind the length: zeros, next to infinities too
            put_row32<T>(smem, r, col, y);                         // dy's place: its last products are done
        }
        fence_async_smem();
        group_sync<kWork>(1);
        if (!maps.rows) {
            store_tile<T, DM, kWork>(smem, [&](int rr) { return seq_row<T>(a.dq, a, s, h, R0 + rr); }, rows - R0, a.D, tid);
        } else if (tid == 0) {
#pragma unroll
            for (int p = 0; p < DM / 64; ++p) tma_store_4d(&maps.dq_rows, base_at + p * kPanel, 64 * p, h * a.G, R0 / a.G, s.b);
            tma_stores_read();
        }
    } else if (warp == kCopier && lane == 0) {
        int issued = 0;
        for (; issued < 2 * kt.count; ++issued) {
            const int slot = issued % S;
            if (issued == S - 1 && !wait_or_stop(smem_u32(&q_moved), 0, stop)) break;
            if (!wait_or_stop(smem_u32(&kv_empty[slot]), ((issued / S) & 1) ^ 1, stop)) break;
            const uint32_t bar = smem_u32(&kv_full[slot]), dst = kv_at + slot * TILE;
            mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
            for (int p = 0; p < DM / 64; ++p)
                tma_load_4d(dst + p * kPanel, issued & 1 ? &maps.v : &maps.k, 64 * p, kt.key(issued >> 1, 128), h, s.b, bar);
            if (issued == 1 && maps.rows) {
                // CTAs start together, and all of them wait for memory then; the rows of the one that follows on this SM come into
                // L2 while this one computes (512 -> 497 us at 2 x 16384 tokens).
                const int64_t id = blockIdx.x + gridDim.x * (h + (int64_t)a.Hkv * blockIdx.z) + maps.sms;
                const int64_t hb = id / gridDim.x;
                const int hn = (int)(hb % a.Hkv), b = (int)(hb / a.Hkv), Rn = (int)(gridDim.x - 1 - id % gridDim.x) * 128;
                if (b < a.B && Rn / a.G < dense_seq(a, b).n) {
#pragma unroll
                    for (int p = 0; p < DM / 64; ++p) {
                        tma_prefetch_4d(&maps.q_rows, 64 * p, hn * a.G, Rn / a.G, b);
                        tma_prefetch_4d(&maps.dy_rows, 64 * p, hn * a.G, Rn / a.G, b);
                        tma_prefetch_4d(&maps.y_rows, 64 * p, hn * a.G, Rn / a.G, b);
                        if (a.rest.data) tma_prefetch_4d(&maps.rest_rows, 64 * p, hn * a.G, Rn / a.G, b);
                    }
                }
            }
        }
        mbar_wait(smem_u32(&q_full), 0, 1u << 12);             // copies in flight land before the memory goes away
        for (int i = max(0, issued - S); i < issued; ++i) mbar_wait(smem_u32(&kv_full[i % S]), (i / S) & 1, 1u << 12);
    } else if (warp == kIssuer && kt.count) {
        const uint32_t lead = elect_one();
        const uint64_t dy_desc = desc_features(base_at), f_desc = desc_features(kv_at), r_desc = desc_rows(kv_at);
        // Waits for the keys and values of tile i, and for `bar`.  A check costs this warp 130 cycles in which no product starts,
        // so its lanes check all three at once.
        auto ready = [&](uint32_t i, uint64_t* bar, uint32_t parity) {
            const uint32_t item = 2 * i + lane;
            return warp_wait(lane < 2 ? smem_u32(&kv_full[item % S]) : smem_u32(bar), lane < 2 ? (item / S) & 1 : parity, stop);
        };
        auto scores = [&](uint32_t i) {
            fence_after();
            mma_dot_ts<DM>(lead, tmem, q_col, f_desc + (2 * i) % S * (TILE >> 4), IDESC_S);
            mma_commit(lead, smem_u32(&s_full));
        };
        auto dprobs = [&](uint32_t i) {
            const uint32_t vs = (2 * i + 1) % S;
            fence_after();
            mma_dot<DM>(lead, tmem + 128, dy_desc, f_desc + vs * (TILE >> 4), IDESC_S);
            mma_commit(lead, smem_u32(&dp_full));
            mma_commit(lead, smem_u32(&kv_empty[vs]));
        };
        const uint32_t count = kt.count;
        bool ok = ready(0, &q_moved, 0);
        if (ok) {
            scores(0);
            dprobs(0);
        }
        for (uint32_t i = 0; i < count && ok; ++i) {
            if (i + 1 < count) {
                if (!(ok = ready(i + 1, &s_free, i & 1))) break;
                scores(i + 1);
                if (!(ok = warp_wait(smem_u32(&dp_free), i & 1, stop))) break;
                dprobs(i + 1);
            }
            if (!(ok = warp_wait(smem_u32(&ds_full), i & 1, stop))) break;
            fence_after();
            const uint32_t ks = (2 * i) % S;
            mma_weighted<128>(lead, o_col, tmem + 256, r_desc + ks * (TILE >> 4), IDESC_O, i != 0);
            mma_commit(lead, smem_u32(&kv_empty[ks]));
            mma_commit(lead, smem_u32(&dq_done));
        }
        mma_commit(lead, smem_u32(ok ? &o_full : &drained));
        if (!ok) mbar_wait(smem_u32(&drained), 0, 1u << 14);   // products in flight end before tensor memory is freed
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kIssuer) tmem_free(tmem, 512);
    if (tid == 0 && stop_flag) report_stop(maps.timeouts, a.status);
}

// ---------------------------------------------------------------- dk, dv
// The steps of a key tile: token tiles outside, query heads of the group inside.
struct Steps {
    int q0, g;
    __device__ __forceinline__ Steps(const SeqArgs& a, int t_lo, int first) : q0(t_lo + first / a.G * 128), g(first % a.G) {}
    __device__ __forceinline__ void next(const SeqArgs& a) {
        if (++g == a.G) g = 0, q0 += 128;
    }
};

// Tiles are transposed: lanes are the CTA's 128 keys, columns 128 tokens of one query head.  Tensor memory: scores 0..127, dP
// 128..255, dv from 256, dk behind it.  The order of the products keeps them running: dv(i), scores(i+1), dk(i), dP(i+1);
// the weights of i + 1 are made during the last two, dS(i) during the first two.
//
// Keys that stay visible to every later token would give their CTA all queries of the sequence; the queries of such tiles are
// dealt to `segments` CTAs, which store Float32 parts for join_kernel to add up in order.
template <typename T, int DM, int FORM>
__global__ void __launch_bounds__(kThreads, 1) umma_dkdv_kernel(const __grid_constant__ SeqArgs a, const __grid_constant__ BwdMaps maps) {
    constexpr int S = kSlots<DM>;
    constexpr uint32_t TILE = kTileBytes<DM>;
    constexpr uint32_t IDESC_S = instr_desc(kIsBf16<T>, 128, false), IDESC_O = instr_desc(kIsBf16<T>, DM, true);
    extern __shared__ char raw[];
    __shared__ uint64_t q_full[S], q_empty[S], kv_full, s_full, dp_full, p_full[2], ds_full[2], st_full[2], st_empty[2], dl_full, dl_empty, o_full, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int stop_flag;
    __shared__ __align__(16) float s_lse[2][128], s_delta[128];       // delta once: the tiles take all but 2 KB
    volatile int* stop = &stop_flag;
    const uint32_t raw_at = smem_u32(raw), base_at = (raw_at + 1023) & ~1023u;
    char* const smem = raw + (base_at - raw_at);
    const uint32_t ring_at = base_at + 2 * TILE;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    __shared__ int ranked;
    const bool rank = FORM && maps.ranked;                         // spans: no first tokens, nothing is dealt out
    const Place place = rank ? place_by_rank() : Place{(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z};
    const int h = place.h, x = place.x;
    const Seq s = dense_seq(a, place.b);
    const int dealt = maps.split_tiles * maps.segments;
    const bool split = x < dealt;
    int tile = split ? x / maps.segments : maps.split_tiles + x - dealt;
    if (rank)
        tile = ranked_tile(gridDim.x, x, reinterpret_cast<int*>(smem + 2 * TILE), &ranked, [&](int first, int last) {
            return first * 128 >= s.n ? 0 : seen_by(a, s, min(last * 128 + 127, s.n - 1)).hi - max(0, seen_by(a, s, first * 128).lo);
        });
    const int seg = split ? x % maps.segments : 0;
    const int k0 = tile * 128;
    int t_lo = max(0, k0 - a.right);                               // queries that see any of the keys
    int t_hi = k0 >= s.n ? t_lo : k0 < a.sinks ? s.n : (int)min((int64_t)s.n, (int64_t)k0 + 128 + a.left);
    int whole_lo = k0 + 127 - a.right, whole_hi = k0 + 127 < a.sinks ? INT_MAX : k0 + a.left;      // that see all of them
    const bool spans = FORM && a.form.spans && k0 < s.n;
    if (FORM && spans) {                                           // neither end of what sees a key falls from one key to the next
        const Reach by0 = seen_by(a, s, k0), by1 = seen_by(a, s, min(k0 + 127, s.n - 1));
        t_lo = max(0, min(by0.lo, k0));
        t_hi = max(k0, min(by1.hi, s.n - 1)) + 1;
        whole_lo = by1.lo;
        whole_hi = by0.hi;
    }
    const int all = max(0, t_hi - t_lo + 127) / 128 * a.G;          // steps: token tiles outside, query heads inside
    const int first = split ? (int)((int64_t)all * seg / maps.segments) : 0;
    const int count = (split ? (int)((int64_t)all * (seg + 1) / maps.segments) : all) - first;

    if (warp == kCopier && lane == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); }
        mbar_init(&kv_full, 1);
        mbar_init(&s_full, 1);
        mbar_init(&dp_full, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&p_full[i], kWarps);
            mbar_init(&ds_full[i], kWarps);
            mbar_init(&st_full[i], 1);
            mbar_init(&st_empty[i], kWarps);
        }
        mbar_init(&dl_full, 1);
        mbar_init(&dl_empty, kWarps);
        mbar_init(&o_full, 1);
        mbar_init(&drained, 1);
        stop_flag = 0;
        mbar_fence_init();
        fence_async_smem();
        if (count) {                                           // on their way while the rest is set up
            mbar_arrive_expect_tx(smem_u32(&kv_full), 2 * TILE);
#pragma unroll
            for (int p = 0; p < DM / 64; ++p) {
                tma_load_4d(base_at + p * kPanel, &maps.k, 64 * p, k0, h, s.b, smem_u32(&kv_full));
                tma_load_4d(base_at + TILE + p * kPanel, &maps.v, 64 * p, k0, h, s.b, smem_u32(&kv_full));
            }
        }
        prefetch_map(&maps.q);
        prefetch_map(&maps.dy);
    }
    if (warp == kIssuer) tmem_alloc(smem_u32(&tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot, dv_col = tmem + 256, dk_col = tmem + 256 + DM;
    // At 64 features the weights and dS have columns of their own; at 128 they overlay what they are made of, and the products of
    // one shape (all 128 x 128 x 16 there) are carried out in the order of their issue.
    const uint32_t p_col = DM == 64 ? tmem + 384 : tmem, ds_col = p_col + (DM == 64 ? 64 : 128), apart = DM == 64 ? 8 : 16;
    float c = 1.f;                                                  // factor of dS
    if (!kIsBf16<T> && count) {
        const int tiles = (int)(((int64_t)s.T * a.G + 127) / 128);
        const float* p = maps.dy_peak + ((int64_t)s.b * a.Hkv + h) * tiles;
        float peak = 0.f;
        for (int i = (int)((int64_t)t_lo * a.G / 128) + lane; i <= (int)(((int64_t)t_hi * a.G - 1) / 128); i += 32) peak = fmaxf(peak, p[i]);
        // keys that the queries t_lo .. t_hi - 1 see: their windows, and first tokens before those
        const float* pv = maps.v_peak + ((int64_t)s.b * a.Hkv + h) * ((a.N + 127) / 128);
        const int from = max(0, reach<FORM>(a, s, t_lo).lo) / 128, upto = min(s.n - 1, reach<FORM>(a, s, t_hi - 1).hi) / 128;
        float v_peak = 0.f;
        for (int i = lane; i <= upto; i += 32)
            if (i >= from || i * 128 < a.sinks) v_peak = fmaxf(v_peak, pv[i]);
        c = ds_factor(warp_max(peak), warp_max(v_peak));
    }

    if (warp < kWarps) {
        const int u = warp >> 2, r = tid & 127, j = k0 + r;
        const uint32_t lane_off = (uint32_t)(warp & 3) << 21;
        const uint32_t S_at = tmem + 16 * u + lane_off, dp_at = S_at + 128, P_at = p_col + apart * u + lane_off, ds_at = ds_col + apart * u + lane_off;
        const f32x2 sc2 = pack2(a.scale_log2, a.scale_log2);
        const float dp_factor = (has_cap(FORM) ? -1.f : 1.f) * (kIsBf16<T> ? 1.f : c / kPScale);
        const f32x2 c2 = pack2(dp_factor, dp_factor);
        const CapPoly<T> poly(a, a.form.cap_in, 1.f);
        const float factor = has_cap(FORM) ? a.form.cap_out : a.scale_log2;
        const bool key_pads = k0 < s.n && mixed<FORM>(a, s, k0, k0 + 127);
        int by_lo = j - a.right, by_hi = j < a.sinks ? s.n - 1 : min(j + a.left, s.n - 1);      // queries that see the key
        if (FORM && spans) {
            const Reach by = seen_by(a, s, j);
            by_lo = by.lo;
            by_hi = min(by.hi, s.n - 1);
        }
        bool ok = true;
        Steps at(a, t_lo, first);
        for (int i = 0; i < count; ++i, at.next(a)) {
            const int q0 = at.q0, b = i & 1;
            const bool pads = FORM && !(q0 >= whole_lo && q0 + 127 <= whole_hi) && mixed<FORM>(a, s, q0, q0 + 127);
            const bool ragged = q0 + 127 >= s.n || k0 + 127 >= s.n || pads || key_pads;
            const bool edge = !(whole_lo <= q0 && q0 + 127 <= whole_hi && q0 + 127 < s.n && k0 + 127 < s.n);
            const float slope = has_slopes(FORM) ? slope_of(a, h * a.G + at.g) : 0.f;
            if (!warp_wait(smem_u32(&st_full[b]), (i >> 1) & 1, stop) || !warp_wait(smem_u32(&s_full), i & 1, stop)) { ok = false; break; }
            fence_after();
            // Columns 16 u .. 16 u + 15 of either half of the tile: the product with the first half starts while the weights
            // of the second are made.
            uint32_t x[kCols], mk = ~0u;
            read_halves(S_at, x);
            if (edge) {
                const int hi = j >= s.n ? -1 : by_hi - q0 - 16 * u, lo = by_lo - q0 - 16 * u;
                mk = (seen_bits(lo, hi, INT_MIN + 1) & 0xffffu) | seen_bits(lo - 64, hi - 64, INT_MIN + 1) << 16;
            }
            if (ragged && u < 2 && (q0 + 127 >= s.n || pads)) { // queries behind the length, and padding, may be anything: zeros
                const int slot = (2 * i + u) % S;               // one warpgroup clears q, another dy
                if (!warp_wait(smem_u32(&q_full[slot]), ((2 * i + u) / S) & 1, stop)) { ok = false; break; }
                if (q0 + r >= s.n || (pads && padding<FORM>(a, s, q0 + r))) clear_row<DM>(smem + (2 + slot) * TILE, r);
                fence_async_smem();
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float4* lse4 = reinterpret_cast<const float4*>(&s_lse[b][64 * g + 16 * u]);
                uint32_t* const xg = x + 16 * g;
                f32x2 inner[has_cap(FORM) ? 8 : 1];
                if (has_cap(FORM)) {
                    if (edge) clear_unseen<16>(xg, mk >> 16 * g);
                    if (FORM == kCap) poly.template scores<16>(xg);
                    else cap_scores<T, 16>(xg, a.form.cap_in, 1.f);
                    cap_inner<16>(inner, xg);
                }
                if (has_slopes(FORM))
                    slope_scores<16>(xg, factor, slope, (float)(j - q0 - 64 * g - 16 * u), k0 + 127 <= q0 ? -1 : q0 + 127 <= k0 ? 1 : 0);
                const f32x2 f2 = has_slopes(FORM) ? pack2(1.f, 1.f) : has_cap(FORM) ? pack2(factor, factor) : sc2;
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 z = lse4[c >> 2];
                    float e[4];
                    unpack2(fma2(pack2(__uint_as_float(xg[c]), __uint_as_float(xg[c + 1])), f2, pack2(z.x, z.y)), e[0], e[1]);
                    unpack2(fma2(pack2(__uint_as_float(xg[c + 2]), __uint_as_float(xg[c + 3])), f2, pack2(z.z, z.w)), e[2], e[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) xg[c + k] = __float_as_uint(fast_exp2(e[k]));
                }
                if (edge) clear_unseen<16>(xg, mk >> 16 * g);
                uint32_t w[8];
#pragma unroll
                for (int c = 0; c < 16; c += 2) w[c >> 1] = pack16<T>(__uint_as_float(xg[c]), __uint_as_float(xg[c + 1]));
                if (has_cap(FORM)) {                               // dS has the cap's derivative
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        float e0, e1;
                        unpack2(mul2(pack2(__uint_as_float(xg[c]), __uint_as_float(xg[c + 1])), inner[c / 2]), e0, e1);
                        xg[c] = __float_as_uint(e0);
                        xg[c + 1] = __float_as_uint(e1);
                    }
                }
                tmem_st8(P_at + 4 * apart * g, w);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[g]));
            }
            if (lane == 0) mbar_arrive(smem_u32(&st_empty[b]));
            if (!warp_wait(smem_u32(&dl_full), i & 1, stop) || !warp_wait(smem_u32(&dp_full), i & 1, stop)) { ok = false; break; }
            fence_after();
            uint32_t y[kCols];
            read_halves(dp_at, y);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float4* del4 = reinterpret_cast<const float4*>(&s_delta[64 * g + 16 * u]);
                uint32_t *const xg = x + 16 * g, *const yg = y + 16 * g;
#pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 z = del4[c >> 2];
                    float e[4];
                    unpack2(mul2(fma2(pack2(__uint_as_float(yg[c]), __uint_as_float(yg[c + 1])), c2, pack2(z.x, z.y)), pack2(__uint_as_float(xg[c]), __uint_as_float(xg[c + 1]))), e[0], e[1]);
                    unpack2(mul2(fma2(pack2(__uint_as_float(yg[c + 2]), __uint_as_float(yg[c + 3])), c2, pack2(z.z, z.w)), pack2(__uint_as_float(xg[c + 2]), __uint_as_float(xg[c + 3]))), e[2], e[3]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) yg[c + k] = __float_as_uint(e[k]);
                }
                if (ragged) clear_unseen<16>(yg, mk >> 16 * g);     // dP of such pairs may be anything
                uint32_t w[8];
#pragma unroll
                for (int c = 0; c < 16; c += 2) w[c >> 1] = pack16<T>(__uint_as_float(yg[c]), __uint_as_float(yg[c + 1]));
                tmem_st8(ds_at + 4 * apart * g, w);
                tmem_wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ds_full[g]));
            }
            if (lane == 0) mbar_arrive(smem_u32(&dl_empty));
        }
        if (count && ok) ok = warp_wait(smem_u32(&o_full), 0, stop);
        fence_after();
        const int which = u & 1;                                   // even warpgroups store dv, odd ones dk, each half of the features
        const float f = !ok || *stop ? __int_as_float(0x7fffffff) : which ? a.scale / c : kIsBf16<T> ? 1.f : 1.f / kPScale;
        float* part = maps.partial + (((((int64_t)s.b * a.Hkv + h) * maps.split_tiles + tile) * maps.segments + seg) * 2 + 1 - which) * (DM * 128) + r;
        char* const stage = smem + which * TILE;                       // the keys' and values' place
#pragma unroll 1
        for (int col = (u >> 1) * (DM / 2); col < ((u >> 1) + 1) * (DM / 2); col += 32) {
            uint32_t o[32];
            tmem_ld32((which ? dk_col : dv_col) + lane_off + col, o);
            tmem_wait_ld();
            settled32(o);
            float y[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) y[e] = count && j < s.n ? __uint_as_float(o[e]) * f : 0.f * f;
            if (split) {
#pragma unroll
                for (int e = 0; e < 32; ++e) part[(col + e) * 128] = y[e];
            } else {
                put_row32<T>(stage, r, col, y);
            }
        }
        if (!split) {
            fence_async_smem();
            group_sync<kWork / 2>(2 + which);
            if (u < 2 && r == 0) {
#pragma unroll
                for (int p = 0; p < DM / 64; ++p) tma_store_4d(which ? &maps.dk : &maps.dv, smem_u32(stage) + p * kPanel, 64 * p, k0, h, s.b);
                tma_stores_read();
            }
        }
    } else if (warp == kCopier && lane == 0 && count) {
        int issued = 0;
        Steps at(a, t_lo, first);
        for (; issued < 2 * count; ++issued) {
            const int slot = issued % S;
            if (!wait_or_stop(smem_u32(&q_empty[slot]), ((issued / S) & 1) ^ 1, stop)) break;
            const uint32_t bar = smem_u32(&q_full[slot]), dst = ring_at + slot * TILE;
            mbar_arrive_expect_tx(bar, TILE);
#pragma unroll
            for (int p = 0; p < DM / 64; ++p)
                tma_load_4d(dst + p * kPanel, issued & 1 ? &maps.dy : &maps.q, 64 * p, at.q0, h * a.G + at.g, s.b, bar);
            if (issued & 1) at.next(a);
        }
        mbar_wait(smem_u32(&kv_full), 0, 1u << 12);            // copies in flight land before the memory goes away
        for (int i = max(0, issued - S); i < issued; ++i) mbar_wait(smem_u32(&q_full[i % S]), (i / S) & 1, 1u << 12);
    } else if (warp == kIssuer && count) {
        const uint32_t lead = elect_one();
        const uint64_t k_desc = desc_features(base_at), v_desc = desc_features(base_at + TILE), f_desc = desc_features(ring_at), r_desc = desc_rows(ring_at);
        const uint32_t steps = count;
        uint32_t have = 0;                                     // queries and cotangents land in order: each is waited for once
        auto landed = [&](uint32_t items) {
            for (; have < items; ++have)
                if (!warp_wait(smem_u32(&q_full[have % S]), (have / S) & 1, stop)) return false;
            return true;
        };
        auto scores = [&](uint32_t i) {
            mma_dot<DM>(lead, tmem, k_desc, f_desc + (2 * i) % S * (TILE >> 4), IDESC_S);
            mma_commit(lead, smem_u32(&s_full));
        };
        auto weighted = [&](uint32_t to, uint32_t from, uint64_t* full, uint32_t slot, uint32_t i) {
#pragma unroll
            for (uint32_t g = 0; g < 2; ++g) {
                if (!warp_wait(smem_u32(&full[g]), i & 1, stop)) return false;
                fence_after();
#pragma unroll
                for (uint32_t k = 4 * g; k < 4 * g + 4; ++k)
                    mma_ts(lead, to, from + k * apart, r_desc + slot * (TILE >> 4) + k * 128, IDESC_O, i != 0 || k != 0);
            }
            return true;
        };
        auto dprobs = [&](uint32_t i) {
            mma_dot<DM>(lead, tmem + 128, v_desc, f_desc + (2 * i + 1) % S * (TILE >> 4), IDESC_S);
            mma_commit(lead, smem_u32(&dp_full));
        };
        bool ok = warp_wait(smem_u32(&kv_full), 0, stop) && landed(2);
        fence_after();
        if (ok) {
            scores(0);
            dprobs(0);
        }
        for (uint32_t i = 0; i < steps && ok; ++i) {
            const uint32_t qs = (2 * i) % S, ds = (2 * i + 1) % S;
            const bool more = i + 1 < steps;
            if (!(ok = (!more || landed(2 * i + 3)) && weighted(dv_col, p_col, p_full, ds, i))) break;
            mma_commit(lead, smem_u32(&q_empty[ds]));
            if (more) scores(i + 1);
            if (!(ok = (!more || landed(2 * i + 4)) && weighted(dk_col, ds_col, ds_full, qs, i))) break;
            mma_commit(lead, smem_u32(&q_empty[qs]));
            if (more) dprobs(i + 1);
        }
        mma_commit(lead, smem_u32(ok ? &o_full : &drained));
        if (!ok) mbar_wait(smem_u32(&drained), 0, 1u << 14);   // products in flight end before tensor memory is freed
    } else if (warp == kFetcher) {
        // minus the rows' sums, and minus their delta, with the factors of half precision
        const float shift = kIsBf16<T> ? 0.f : kPLog2, minus = (has_cap(FORM) ? 1.f : -1.f) * (kIsBf16<T> ? 1.f : c / kPScale);
        const int rows = s.T * a.G;
        const int64_t stat0 = ((int64_t)s.b * a.Hkv + h) * rows;
        Steps at(a, t_lo, first);
        for (int i = 0; i < count; ++i, at.next(a)) {
            const int b = i & 1;
            float z[4], d[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = at.q0 + lane + 32 * k;
                const bool in = t < s.n;
                z[k] = in ? shift - a.lse[stat0 + (int64_t)t * a.G + at.g] : 0.f;
                d[k] = in ? minus * a.delta[stat0 + (int64_t)t * a.G + at.g] : 0.f;
            }
            if (!warp_wait(smem_u32(&st_empty[b]), ((i >> 1) & 1) ^ 1, stop)) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) s_lse[b][lane + 32 * k] = z[k];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&st_full[b]));
            if (!warp_wait(smem_u32(&dl_empty), (i & 1) ^ 1, stop)) break;
#pragma unroll
            for (int k = 0; k < 4; ++k) s_delta[lane + 32 * k] = d[k];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&dl_full));
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kIssuer) tmem_free(tmem, 512);
    if (tid == 0 && stop_flag) report_stop(maps.timeouts, a.status);
}

// Adds the parts of a split key tile in order: thread = key, eight features of dk or dv a block.
template <typename T, int DM>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ SeqArgs a, const float* __restrict__ partial, int split_tiles, int segments) {
    const int r = threadIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int c = blockIdx.x % (DM / 8) * 8, which = blockIdx.x / (DM / 8) & 1, tile = blockIdx.x / (DM / 4), j = tile * 128 + r;
    const float* p = partial + ((((int64_t)b * a.Hkv + h) * split_tiles + tile) * segments * 2 + which) * (DM * 128) + c * 128 + r;
    float sum[8] = {};
#pragma unroll 4
    for (int seg = 0; seg < segments; ++seg, p += 2 * DM * 128)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += p[e * 128];
    if (j >= a.N || c >= a.D) return;
    const ca_seq_view& out = which ? a.dv : a.dk;
    T* dst = (T*)out.data + h * out.head + (int64_t)j * out.token + b * out.batch + c;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack16<T>(sum[0], sum[1]), pack16<T>(sum[2], sum[3]), pack16<T>(sum[4], sum[5]), pack16<T>(sum[6], sum[7]));
}

template <typename T, int DM, int FORM>
int launch(const SeqArgs& a, const BwdMaps& maps, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(umma_dq_kernel<T, DM, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBwdSmem<DM>);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(umma_dkdv_kernel<T, DM, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBwdSmem<DM>);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    if (!kIsBf16<T>) {
        peak_kernel<FORM><<<dim3((a.N + 127) / 128, a.Hkv, a.B), 256, 0, st>>>(a, maps.v_peak);
        CA_CHECK_LAUNCH("window peak kernel");
    }
    umma_dq_kernel<T, DM, FORM><<<dim3((unsigned)(((int64_t)a.N * a.G + 127) / 128), a.Hkv, a.B), kThreads, kBwdSmem<DM>, st>>>(a, maps);
    count_tensor_launch();
    CA_CHECK_LAUNCH("window dq kernel (tensor cores)");
    const int tiles = (a.N + 127) / 128;
    umma_dkdv_kernel<T, DM, FORM><<<dim3(tiles - maps.split_tiles + maps.split_tiles * maps.segments, a.Hkv, a.B), kThreads, kBwdSmem<DM>, st>>>(a, maps);
    count_tensor_launch();
    CA_CHECK_LAUNCH("window dk/dv kernel (tensor cores)");
    if (maps.split_tiles) {
        join_kernel<T, DM><<<dim3(maps.split_tiles * (DM / 4), a.Hkv, a.B), 128, 0, st>>>(a, maps.partial, maps.split_tiles, maps.segments);
        CA_CHECK_LAUNCH("window dk/dv join kernel");
    }
    return CA_OK;
}

}  // namespace

static size_t dy_peaks(const SeqArgs& a) { return ((size_t)a.N * a.G + 127) / 128 * a.Hkv * a.B; }
static size_t peak_floats(const SeqArgs& a) { return (dy_peaks(a) + ((size_t)a.N + 127) / 128 * a.Hkv * a.B + 63) & ~(size_t)63; }

// Behind the rows' delta: the peaks of dy, and the Float32 parts of the dealt key tiles.
size_t umma_bwd_parts(const SeqArgs& a) {
    const Dealt p = deal_first_tokens(a, 128);
    return (peak_floats(a) + (size_t)p.tiles * p.segments * 2 * (a.D > 64 ? 128 : 64) * 128 * a.Hkv * a.B) * sizeof(float);
}

int umma_window_bwd(const SeqArgs& a, int dtype, float* parts, cudaStream_t st) {
    BwdMaps maps{};
    const bool bf16 = dtype == CA_BF16;
    int rc;
    if ((rc = encode_tokens(&maps.k, bf16, a.k, a.D, a.Hkv, a.N, a.B)) || (rc = encode_tokens(&maps.v, bf16, a.v, a.D, a.Hkv, a.N, a.B)) ||
        (rc = encode_tokens(&maps.q, bf16, a.q, a.D, a.Hq, a.N, a.B)) || (rc = encode_tokens(&maps.dy, bf16, a.dy, a.D, a.Hq, a.N, a.B)))
        return rc;
    if ((rc = encode_tokens(&maps.dk, bf16, a.dk, a.D, a.Hkv, a.N, a.B)) || (rc = encode_tokens(&maps.dv, bf16, a.dv, a.D, a.Hkv, a.N, a.B))) return rc;
    maps.rows = rows_fit(a);
    if (maps.rows && ((rc = encode_rows(&maps.q_rows, bf16, a.q, a)) || (rc = encode_rows(&maps.dy_rows, bf16, a.dy, a)) ||
                      (rc = encode_rows(&maps.dq_rows, bf16, a.dq, a)) || (rc = encode_rows(&maps.y_rows, bf16, a.y, a)) ||
                      (a.rest.data && (rc = encode_rows(&maps.rest_rows, bf16, a.rest, a)))))
        return rc;
    maps.sms = sm_count();
    maps.ranked = a.form.spans && (int64_t)((a.N + 127) / 128) * a.Hkv * a.B > maps.sms;      // else all blocks start at once
    if (!(maps.timeouts = stage_timeout_counter())) return cuda_fail(cudaGetLastError(), "cudaGetSymbolAddress(stage timeouts)");
    maps.dy_peak = parts;
    maps.v_peak = parts + dy_peaks(a);
    maps.partial = parts + peak_floats(a);
    const Dealt p = deal_first_tokens(a, 128);
    maps.split_tiles = p.tiles;
    maps.segments = p.segments;
    const bool wide = a.D > 64;
#define CA_BWD(FORM)                                                                                                      \
    return bf16 ? (wide ? launch<__nv_bfloat16, 128, FORM>(a, maps, st) : launch<__nv_bfloat16, 64, FORM>(a, maps, st))   \
                : (wide ? launch<__half, 128, FORM>(a, maps, st) : launch<__half, 64, FORM>(a, maps, st))
    switch (a.kind) {
        case kMasks: CA_BWD(kMasks);
        case kSlopes: CA_BWD(kSlopes);
        case kCap: CA_BWD(kCap);
        case kCapSlopes: CA_BWD(kCapSlopes);
        default: CA_BWD(kNoForm);
    }
#undef CA_BWD
}

}  // namespace ca
