// Attention on token sequences in Float32, on the FMA pipe: dense tensors and a paged cache.
//
// The tensor cores round Float32 operands, so every product is an FMA here, two at a time (fma.rn.f32x2).  Pairs of halves with
// short sums, as the circulant sweeps use them (split.cuh: errors of 2e-7 to 4e-7), are not built for these kernels.
//
// Tiles of 64 rows and 64 columns in shared memory, features fastest and rows padded by 4 floats, so that the 16-byte
// reads of eight lanes (rows 1 apart) fall into different banks.  A thread (ty, tx) of 16 x 16 holds the products of rows
// ty + 16i with columns tx + 16j (i, j < 4): 32 packed FMA for 8 reads of 16 bytes.  The next tile is copied (cp.async)
// while this one is worked on (forward), or another block works (backward: two blocks on an SM with one stage each beat one
// with two, 274 us against 311 for dq).
//
// Bound: shared memory.  A 4 x 4 piece of products takes one 16-byte read for four packed FMA, and reads keep that unit 75 to 83 %
// busy; larger pieces do not fit 128 registers (two blocks an SM) next to the accumulators.  2 x 4096 tokens, 8 heads of 64
// features, window 256: forward 206 us, dq 275, dk and dv 354.  12 chunks of up to 900 tokens over a cache (128 features): 3570 us.
#include "seq.cuh"
#include "umma.cuh"

namespace ca {
namespace {

constexpr int kTile = 64, kThreads = 256, kPPitch = kTile + 4;
template <int DM> constexpr int kPitch = DM + 4;
template <int DM> constexpr int kTileFloats = kTile * kPitch<DM>;

__device__ __forceinline__ void copy16(float* dst, const float* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// 64 rows of D features; `row(r, on)` gives the address of row r and clears `on` where the row counts as zeros.
template <int DM, typename Row>
__device__ __forceinline__ void fetch(float* dst, Row row, const float* any, int D, int tid) {
    constexpr int PIECES = DM / 4, STEP = kThreads / PIECES;
    const int c = tid % PIECES;
#pragma unroll
    for (int r = tid / PIECES; r < kTile; r += STEP) {
        bool on = c * 4 < D;
        const float* src = row(r, on);
        copy16(dst + r * kPitch<DM> + c * 4, on ? src + c * 4 : any, on);
    }
}

// s[i][j] = row ty+16i of A times row tx+16j of B.
template <int DM>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float (&s)[4][4]) {
    constexpr int P = kPitch<DM>;
    f32x2 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0;
#pragma unroll 4
    for (int d = 0; d < DM; d += 4) {
        ulonglong2 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const ulonglong2*)(A + (ty + 16 * i) * P + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *(const ulonglong2*)(B + (tx + 16 * j) * P + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fma2(x[i].y, y[j].y, fma2(x[i].x, y[j].x, acc[i][j]));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float lo, hi;
            unpack2(acc[i][j], lo, hi);
            s[i][j] = lo + hi;
        }
}

// o[i][2c], o[i][2c+1]: += row ty+16i of P times columns (tx*4 + 64*(c/2) + 2*(c%2)) and the next pair of B.
template <int DM>
__device__ __forceinline__ void acc_tile(const float* Pm, const float* B, int ty, int tx, f32x2 (&o)[4][DM / 32]) {
    constexpr int P = kPitch<DM>;
#pragma unroll 2
    for (int k = 0; k < kTile; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *(const float4*)(Pm + (ty + 16 * i) * kPPitch + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            f32x2 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
                w[i] = pack2(e, e);
            }
#pragma unroll
            for (int c = 0; c < DM / 64; ++c) {
                const ulonglong2 v = *(const ulonglong2*)(B + (k + kk) * P + tx * 4 + 64 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i][2 * c] = fma2(w[i], v.x, o[i][2 * c]);
                    o[i][2 * c + 1] = fma2(w[i], v.y, o[i][2 * c + 1]);
                }
            }
        }
    }
}

__device__ __forceinline__ float max16(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
    for (int o = 8; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

template <int DM>
__device__ __forceinline__ void clear_row(f32x2 (&o)[DM / 32]) {
#pragma unroll
    for (int c = 0; c < DM / 32; ++c) o[c] = 0;
}

template <int DM>
__device__ __forceinline__ void store_row(float* dst, const f32x2 (&o)[DM / 32], float f, int D, int tx) {
    const f32x2 f2 = pack2(f, f);
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
        const int at = tx * 4 + 64 * c;
        if (at >= D) continue;
        ulonglong2 w;
        w.x = mul2(o[2 * c], f2);
        w.y = mul2(o[2 * c + 1], f2);
        *(ulonglong2*)(dst + at) = w;
    }
}

__device__ __forceinline__ float* row_ptr(const ca_seq_view& v, const SeqArgs& a, const Seq& s, int h, int R) {
    const int t = token_of(a, R), g = R - t * a.G;
    return (float*)v.data + (h * a.G + g) * v.head + (int64_t)(s.t0 + t) * v.token + (a.pages.table ? 0 : s.b * v.batch);
}
// Key row j; clears `on` where it does not exist.
__device__ __forceinline__ const float* key_ptr(const ca_seq_view& v, const ca_page_view& pv, const SeqArgs& a, const Seq& s, int h, int j, bool& on) {
    on = on && j < s.n;
    if (!a.pages.table) return (const float*)v.data + h * v.head + (int64_t)j * v.token + s.b * v.batch;
    const int p = on ? page_of(a, s.b, j) : -1;
    on = on && p >= 0;
    return (const float*)pv.data + h * pv.head + (int64_t)(j % a.pages.page) * pv.token + p * pv.page;
}

// ---------------------------------------------------------------- forward
template <int DM> constexpr size_t kFwdSmem = (5 * kTileFloats<DM> + kTile * kPPitch) * sizeof(float);

template <int DM>
__global__ void __launch_bounds__(kThreads) fma_fwd_kernel(const __grid_constant__ SeqArgs a) {
    extern __shared__ float4 smem4[];
    float *Q = (float*)smem4, *KV = Q + kTileFloats<DM>, *Pm = KV + 4 * kTileFloats<DM>;      // K, V, K, V
    __shared__ unsigned char gone[2][kTile];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y;
    int tile = blockIdx.x;
    int2 owned;
    Seq s;
    if (a.pages.table) {
        owned = owned_tokens(a);
        if (!paged_seq(a, kTile, tile, &s)) {
            clear_unowned<float>(a, owned, h, tid, kThreads);
            return;
        }
    } else {
        s = dense_seq(a, blockIdx.z);
    }
    const int rows = s.T * a.G, R0 = tile * kTile;
    const int p_lo = s.base + R0 / a.G, p_hi = s.base + (min(R0 + kTile, rows) - 1) / a.G;
    const float* any = (const float*)a.q.data;
    fetch<DM>(Q, [&](int r, bool& on) {
        const int R = min(R0 + r, rows - 1), pos = s.base + token_of(a, R);
        on = on && R0 + r < rows && pos >= 0 && pos < s.n;
        return row_ptr(a.q, a, s, h, R);
    }, any, a.D, tid);
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, kTile);
    auto prefetch = [&](int it) {
        const int j0 = kt.key(it, kTile), b = it & 1;
        float* K = KV + 2 * b * kTileFloats<DM>;
        fetch<DM>(K, [&](int r, bool& on) {
            const bool whole = on;
            const float* p = key_ptr(a.k, a.kp, a, s, h, j0 + r, on);
            if (tid % (DM / 4) == 0 && whole) gone[b][r] = !on;
            return p;
        }, any, a.D, tid);
        // rows of v that no query of this tile sees may hold anything: they count as zeros
        fetch<DM>(K + kTileFloats<DM>, [&](int r, bool& on) {
            const int j = j0 + r;
            on = on && (j >= p_lo - a.left || j < a.sinks) && j <= (int64_t)p_hi + a.right;
            return key_ptr(a.v, a.vp, a, s, h, j, on);
        }, any, a.D, tid);
    };
    int pos[4];
    float m[4], l[4];
    f32x2 o[4][DM / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int R = R0 + ty + 16 * i;
        pos[i] = R < rows ? s.base + token_of(a, R) : -1;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DM / 32; ++c) o[i][c] = 0;
    }
    if (kt.count) prefetch(0);
    copies_commit();
    if (a.pages.table) clear_unowned<float>(a, owned, h, tid, kThreads);
    for (int it = 0; it < kt.count; ++it) {
        if (it + 1 < kt.count) prefetch(it + 1);
        copies_commit();
        copies_wait<1>();
        __syncthreads();
        const int j0 = kt.key(it, kTile), b = it & 1;
        const float* K = KV + 2 * b * kTileFloats<DM>;
        float sc[4][4];
        dot_tile<DM>(Q, K, ty, tx, sc);
        const bool edge = !(p_lo >= 0 && p_hi < s.n && j0 + kTile - 1 <= (int64_t)p_lo + a.right && j0 + kTile <= s.n &&
                            (j0 >= p_hi - a.left || j0 + kTile <= a.sinks)) || a.pages.table;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sc[i][j] *= a.scale_log2;
                if (edge && (!sees(a, s.n, pos[i], j0 + tx + 16 * j) || gone[b][tx + 16 * j])) sc[i][j] = -INFINITY;
                top = fmaxf(top, sc[i][j]);
            }
            top = max16(top);
            const float ref = top == -INFINITY ? 0.f : top;       // a row that has seen nothing yet
            const float f = fast_exp2(m[i] - ref);
            m[i] = top;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = fast_exp2(sc[i][j] - ref);
                sum += p;
                Pm[(ty + 16 * i) * kPPitch + tx + 16 * j] = p;
            }
            l[i] = l[i] * f + sum;
            const f32x2 f2 = pack2(f, f);
#pragma unroll
            for (int c = 0; c < DM / 32; ++c) o[i][c] = mul2(o[i][c], f2);
        }
        __syncwarp();                                             // rows ty + 16i are written and read by one half warp
        acc_tile<DM>(Pm, K + kTileFloats<DM>, ty, tx, o);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int R = R0 + ty + 16 * i;
        const float sum = sum16(l[i]);
        if (R >= rows) continue;
        if (sum == 0.f) clear_row<DM>(o[i]);                          // sees nothing: zeros, next to infinities too
        store_row<DM>(row_ptr(a.y, a, s, h, R), o[i], sum > 0.f ? 1.f / sum : 0.f, a.D, tx);
        if (a.lse && tx == 0) a.lse[((int64_t)s.b * a.Hkv + h) * rows + R] = sum > 0.f ? m[i] + log2f(sum) : -INFINITY;
    }
}

// ---------------------------------------------------------------- backward
// P = 2^(scale q.k log2 e - lse), dP = dy.v, dS = P (dP - delta), delta = dy.y; dq = scale dS k.
template <int DM> constexpr size_t kDqSmem = (4 * kTileFloats<DM> + kTile * kPPitch) * sizeof(float);

template <int DM>
__global__ void __launch_bounds__(kThreads, DM == 64 ? 2 : 1) fma_dq_kernel(const __grid_constant__ SeqArgs a) {
    extern __shared__ float4 smem4[];
    float *Q = (float*)smem4, *O = Q + kTileFloats<DM>, *K = O + kTileFloats<DM>, *V = K + kTileFloats<DM>, *Pm = V + kTileFloats<DM>;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y;
    const Seq s = dense_seq(a, blockIdx.z);
    const int rows = s.T * a.G, R0 = blockIdx.x * kTile;
    const int p_lo = R0 / a.G, p_hi = (min(R0 + kTile, rows) - 1) / a.G;
    const int64_t stat0 = ((int64_t)s.b * a.Hkv + h) * rows;
    const float* any = (const float*)a.q.data;
    auto from = [&](const ca_seq_view& v) {
        return [&](int r, bool& on) {
            const int R = min(R0 + r, rows - 1);
            on = on && R0 + r < rows && token_of(a, R) < s.n;
            return (const float*)row_ptr(v, a, s, h, R);
        };
    };
    fetch<DM>(Q, from(a.q), any, a.D, tid);
    fetch<DM>(O, from(a.dy), any, a.D, tid);
    float* yrow = V;                                              // y passes through the values' place
    fetch<DM>(yrow, from(a.y), any, a.D, tid);
    copies_commit();
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, kTile);
    auto prefetch = [&](int it) {
        const int j0 = kt.key(it, kTile);
        fetch<DM>(K, [&](int r, bool& on) { return key_ptr(a.k, a.kp, a, s, h, j0 + r, on); }, any, a.D, tid);
        fetch<DM>(V, [&](int r, bool& on) { return key_ptr(a.v, a.vp, a, s, h, j0 + r, on); }, any, a.D, tid);
    };
    copies_wait<0>();
    __syncthreads();
    int pos[4];
    float lse[4], delta[4];
    f32x2 o[4][DM / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i, R = R0 + r;
        float d = 0.f;
        for (int f = tx; f < DM; f += 16) d = fmaf(O[r * kPitch<DM> + f], yrow[r * kPitch<DM> + f], d);
        delta[i] = sum16(d);
        pos[i] = R < rows ? token_of(a, R) : -1;
        lse[i] = R < rows ? a.lse[stat0 + R] : 0.f;
        if (R < rows && tx == 0) a.delta[stat0 + R] = delta[i];
#pragma unroll
        for (int c = 0; c < DM / 32; ++c) o[i][c] = 0;
    }
    __syncthreads();
    for (int it = 0; it < kt.count; ++it) {
        prefetch(it);
        copies_commit();
        copies_wait<0>();
        __syncthreads();
        const int j0 = kt.key(it, kTile);
        const bool edge = !(p_hi < s.n && j0 + kTile - 1 <= (int64_t)p_lo + a.right && j0 + kTile <= s.n && (j0 >= p_hi - a.left || j0 + kTile <= a.sinks));
        float sc[4][4], dp[4][4];
        dot_tile<DM>(Q, K, ty, tx, sc);
        dot_tile<DM>(O, V, ty, tx, dp);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool see = !edge || sees(a, s.n, pos[i], j0 + tx + 16 * j);
                Pm[(ty + 16 * i) * kPPitch + tx + 16 * j] = see ? fast_exp2(sc[i][j] * a.scale_log2 - lse[i]) * (dp[i][j] - delta[i]) : 0.f;
            }
        __syncwarp();
        acc_tile<DM>(Pm, K, ty, tx, o);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int R = R0 + ty + 16 * i;
        if (pos[i] >= s.n) clear_row<DM>(o[i]);
        if (R < rows) store_row<DM>(row_ptr(a.dq, a, s, h, R), o[i], a.scale, a.D, tx);
    }
}

// A block owns 64 keys and walks the query rows that see any of them: dv = P^T dy, dk = scale dS^T q, no atomics.  The rows of
// key tiles that hold first tokens are dealt to `segments` blocks, whose parts fma_join_kernel adds up in order.
template <int DM> constexpr size_t kDkdvSmem = (4 * kTileFloats<DM> + 2 * kTile * kPPitch) * sizeof(float);

struct Parts {
    float* data;            // [b][key head][tile][segment][dk, dv][64 keys][DM]
    int tiles, segments;
};

template <int DM>
__global__ void __launch_bounds__(kThreads, DM == 64 ? 2 : 1) fma_dkdv_kernel(const __grid_constant__ SeqArgs a, const Parts parts) {
    extern __shared__ float4 smem4[];
    float *K = (float*)smem4, *V = K + kTileFloats<DM>, *Q = V + kTileFloats<DM>, *O = Q + kTileFloats<DM>, *Pm = O + kTileFloats<DM>, *Sm = Pm + kTile * kPPitch;
    __shared__ float s_lse[kTile], s_delta[kTile];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y;
    const int dealt = parts.tiles * parts.segments;
    const bool split = (int)blockIdx.x < dealt;
    const int tile = split ? (int)blockIdx.x / parts.segments : parts.tiles + (int)blockIdx.x - dealt, seg = split ? (int)blockIdx.x % parts.segments : 0;
    const int j0 = tile * kTile;
    const Seq s = dense_seq(a, blockIdx.z);
    const int rows = s.T * a.G;
    const int64_t stat0 = ((int64_t)s.b * a.Hkv + h) * rows;
    const float* any = (const float*)a.q.data;
    fetch<DM>(K, [&](int r, bool& on) { return key_ptr(a.k, a.kp, a, s, h, j0 + r, on); }, any, a.D, tid);
    fetch<DM>(V, [&](int r, bool& on) { return key_ptr(a.v, a.vp, a, s, h, j0 + r, on); }, any, a.D, tid);
    f32x2 dk[4][DM / 32], dv[4][DM / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DM / 32; ++c) dk[i][c] = dv[i][c] = 0;
    const int t_lo = max(0, j0 - a.right);
    const int t_hi = j0 >= s.n ? t_lo : j0 < a.sinks ? s.n : (int)min((int64_t)s.n, (int64_t)j0 + kTile + a.left);
    const int lo = t_lo * a.G, hi = max(t_lo, t_hi) * a.G, all = (hi - lo + kTile - 1) / kTile;
    const int first = split ? (int)((int64_t)all * seg / parts.segments) : 0;
    const int count = (split ? (int)((int64_t)all * (seg + 1) / parts.segments) : all) - first;
    auto prefetch = [&](int it) {
        const int R0 = lo + (first + it) * kTile;
        auto from = [&](const ca_seq_view& v) {
            return [&](int r, bool& on) {
                on = on && R0 + r < hi;
                return (const float*)row_ptr(v, a, s, h, min(R0 + r, hi - 1));
            };
        };
        fetch<DM>(Q, from(a.q), any, a.D, tid);
        fetch<DM>(O, from(a.dy), any, a.D, tid);
        if (tid < kTile) {
            const bool have = R0 + tid < hi;
            s_lse[tid] = have ? a.lse[stat0 + R0 + tid] : 0.f;
            s_delta[tid] = have ? a.delta[stat0 + R0 + tid] : 0.f;
        }
    };
    if (count) prefetch(0);
    copies_commit();
    for (int it = 0; it < count; ++it) {
        copies_wait<0>();
        __syncthreads();
        const int R0 = lo + (first + it) * kTile;
        float sc[4][4], dp[4][4];
        dot_tile<DM>(K, Q, ty, tx, sc);
        dot_tile<DM>(V, O, ty, tx, dp);
        const int t0 = R0 / a.G, t1 = min(R0 + kTile, hi) - 1 < R0 ? t0 : (min(R0 + kTile, hi) - 1) / a.G;
        const bool edge = !(R0 + kTile <= hi && t1 < s.n && j0 + kTile <= s.n && j0 + kTile - 1 <= (int64_t)t0 + a.right && (j0 >= t1 - a.left || j0 + kTile <= a.sinks));
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int R = R0 + tx + 16 * c;
                const bool see = !edge || (R < hi && sees(a, s.n, token_of(a, R), j0 + ty + 16 * i));
                const float p = see ? fast_exp2(sc[i][c] * a.scale_log2 - s_lse[tx + 16 * c]) : 0.f;
                Pm[(ty + 16 * i) * kPPitch + tx + 16 * c] = p;
                Sm[(ty + 16 * i) * kPPitch + tx + 16 * c] = see ? p * (dp[i][c] - s_delta[tx + 16 * c]) : 0.f;
            }
        __syncwarp();
        acc_tile<DM>(Pm, O, ty, tx, dv);
        acc_tile<DM>(Sm, Q, ty, tx, dk);
        __syncthreads();
        if (it + 1 < count) prefetch(it + 1);
        copies_commit();
    }
    copies_wait<0>();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i, j = j0 + r;
        if (j >= s.n) {
            clear_row<DM>(dk[i]);
            clear_row<DM>(dv[i]);
        }
        if (split) {
            float* p = parts.data + ((((int64_t)s.b * a.Hkv + h) * parts.tiles + tile) * parts.segments + seg) * 2 * kTile * DM + r * DM;
            store_row<DM>(p, dk[i], a.scale, DM, tx);
            store_row<DM>(p + kTile * DM, dv[i], 1.f, DM, tx);
        } else if (j < a.N) {
            store_row<DM>((float*)a.dk.data + h * a.dk.head + (int64_t)j * a.dk.token + s.b * a.dk.batch, dk[i], a.scale, a.D, tx);
            store_row<DM>((float*)a.dv.data + h * a.dv.head + (int64_t)j * a.dv.token + s.b * a.dv.batch, dv[i], 1.f, a.D, tx);
        }
    }
}

template <int DM>
__global__ void __launch_bounds__(256) fma_join_kernel(const __grid_constant__ SeqArgs a, const Parts parts) {
    const int which = blockIdx.x & 1, piece = blockIdx.x >> 1 & 3, tile = blockIdx.x >> 3, h = blockIdx.y, b = blockIdx.z;
    const float* p = parts.data + (((int64_t)b * a.Hkv + h) * parts.tiles + tile) * parts.segments * 2 * kTile * DM + which * kTile * DM;
    const ca_seq_view& out = which ? a.dv : a.dk;
    for (int i = piece * 256 + threadIdx.x; i < kTile * DM / 4; i += 4 * 256) {
        const int r = i / (DM / 4), c = i % (DM / 4) * 4, j = tile * kTile + r;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int seg = 0; seg < parts.segments; ++seg) {
            const float4 x = *(const float4*)(p + (int64_t)seg * 2 * kTile * DM + r * DM + c);
            sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
        }
        if (j < a.N && c < a.D) *(float4*)((float*)out.data + h * out.head + (int64_t)j * out.token + b * out.batch + c) = sum;
    }
}

template <typename K>
int raise_smem(K kernel, size_t bytes) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? CA_OK : cuda_fail(e, "cudaFuncSetAttribute");
}

template <int DM>
int launch_fwd(const SeqArgs& a, cudaStream_t st) {
    const int rc = raise_smem(fma_fwd_kernel<DM>, kFwdSmem<DM>);
    if (rc) return rc;
    const int64_t tiles = a.pages.table ? paged_tiles(a.N, a.G, a.pages.sequences, kTile) : ((int64_t)a.N * a.G + kTile - 1) / kTile;
    fma_fwd_kernel<DM><<<dim3((unsigned)tiles, a.Hkv, a.B), kThreads, kFwdSmem<DM>, st>>>(a);
    CA_CHECK_LAUNCH("window forward kernel");
    return CA_OK;
}

template <int DM>
int launch_bwd(const SeqArgs& a, float* data, cudaStream_t st) {
    int rc = raise_smem(fma_dq_kernel<DM>, kDqSmem<DM>);
    if (rc || (rc = raise_smem(fma_dkdv_kernel<DM>, kDkdvSmem<DM>))) return rc;
    const Dealt p = deal_first_tokens(a, kTile);
    const Parts parts{data, p.tiles, p.segments};
    fma_dq_kernel<DM><<<dim3((unsigned)(((int64_t)a.N * a.G + kTile - 1) / kTile), a.Hkv, a.B), kThreads, kDqSmem<DM>, st>>>(a);
    CA_CHECK_LAUNCH("window dq kernel");
    const int tiles = (a.N + kTile - 1) / kTile;
    fma_dkdv_kernel<DM><<<dim3(tiles - parts.tiles + parts.tiles * parts.segments, a.Hkv, a.B), kThreads, kDkdvSmem<DM>, st>>>(a, parts);
    CA_CHECK_LAUNCH("window dk/dv kernel");
    if (parts.tiles) {
        fma_join_kernel<DM><<<dim3(8 * parts.tiles, a.Hkv, a.B), 256, 0, st>>>(a, parts);
        CA_CHECK_LAUNCH("window dk/dv join kernel");
    }
    return CA_OK;
}

}  // namespace

size_t fma_bwd_parts(const SeqArgs& a) {
    const Dealt p = deal_first_tokens(a, kTile);
    return (size_t)p.tiles * p.segments * 2 * kTile * (a.D > 64 ? 128 : 64) * a.Hkv * a.B * sizeof(float);
}

int fma_fwd(const SeqArgs& a, cudaStream_t st) { return a.D > 64 ? launch_fwd<128>(a, st) : launch_fwd<64>(a, st); }
int fma_bwd(const SeqArgs& a, float* parts, cudaStream_t st) { return a.D > 64 ? launch_bwd<128>(a, parts, st) : launch_bwd<64>(a, parts, st); }

}  // namespace ca
