// Attention on token sequences on the FMA pipe, in Float32.
//
// Tiles of 64 rows and 64 columns in shared memory, features fastest and rows padded by 4 floats, so that the 16-byte
// reads of eight lanes (rows 1 apart) fall into different banks.  A thread (ty, tx) of 16 x 16 holds the products of rows
// ty + 16i with columns tx + 16j (i, j < 4): 64 FMA for 8 reads of 16 bytes.
#include "seq.cuh"

namespace ca {
namespace {

constexpr int kTile = 64, kThreads = 256, kPPitch = kTile + 4;

template <int DM> constexpr int kPitch = DM + 4;

// One row of D elements -> Float32 in shared memory, zeros behind D and where `src` is null; four threads a row.
template <typename T, int DM>
__device__ __forceinline__ void load_row(float* dst, const T* src, int D, int part) {
#pragma unroll 4
    for (int f = part * 4; f < DM; f += 16) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (src && f < D) {
            if (sizeof(T) == 4) {
                x = *(const float4*)(src + f);
            } else {
                const uint2 w = *(const uint2*)(src + f);
                const T* e = (const T*)&w;
                x = make_float4(to_float(e[0]), to_float(e[1]), to_float(e[2]), to_float(e[3]));
            }
        }
        *(float4*)(dst + f) = x;
    }
}

// s[i][j] = row ty+16i of A times row tx+16j of B.
template <int DM>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float (&s)[4][4]) {
    constexpr int P = kPitch<DM>;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DM; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *(const float4*)(A + (ty + 16 * i) * P + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *(const float4*)(B + (tx + 16 * j) * P + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                s[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, s[i][j]))));
    }
}

// o[i][c] += row ty+16i of P times column (tx*4 + 64*(c/4) + c%4) of B.
template <int DM>
__device__ __forceinline__ void acc_tile(const float* Pm, const float* B, int ty, int tx, float (&o)[4][DM / 16]) {
    constexpr int P = kPitch<DM>;
#pragma unroll 2
    for (int k = 0; k < kTile; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *(const float4*)(Pm + (ty + 16 * i) * kPPitch + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int c = 0; c < DM / 64; ++c) {
                const float4 v = *(const float4*)(B + (k + kk) * P + tx * 4 + 64 * c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
                    o[i][4 * c + 0] = fmaf(w, v.x, o[i][4 * c + 0]);
                    o[i][4 * c + 1] = fmaf(w, v.y, o[i][4 * c + 1]);
                    o[i][4 * c + 2] = fmaf(w, v.z, o[i][4 * c + 2]);
                    o[i][4 * c + 3] = fmaf(w, v.w, o[i][4 * c + 3]);
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

template <typename T, int DM>
__device__ __forceinline__ void store_row(T* dst, const float (&o)[DM / 16], float f, int D, int tx) {
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
        const int at = tx * 4 + 64 * c;
        if (at >= D) continue;
        if (sizeof(T) == 4) {
            *(float4*)(dst + at) = make_float4(o[4 * c] * f, o[4 * c + 1] * f, o[4 * c + 2] * f, o[4 * c + 3] * f);
        } else {
            T e[4] = {from_float<T>(o[4 * c] * f), from_float<T>(o[4 * c + 1] * f), from_float<T>(o[4 * c + 2] * f), from_float<T>(o[4 * c + 3] * f)};
            *(uint2*)(dst + at) = *(const uint2*)e;
        }
    }
}

template <typename T>
__device__ __forceinline__ T* row_ptr(const ca_seq_view& v, const SeqArgs& a, const Seq& s, int h, int R) {
    const int t = R / a.G, g = R - t * a.G;
    return (T*)v.data + (h * a.G + g) * v.head + (int64_t)(s.t0 + t) * v.token + (a.pages.table ? 0 : s.b * v.batch);
}
// Key row j, or null where it does not exist.
template <typename T>
__device__ __forceinline__ const T* key_ptr(const ca_seq_view& v, const ca_page_view& pv, const SeqArgs& a, const Seq& s, int h, int j) {
    if (j >= s.n) return nullptr;
    if (!a.pages.table) return (const T*)v.data + h * v.head + (int64_t)j * v.token + s.b * v.batch;
    const int p = page_of(a, s.b, j);
    return p < 0 ? nullptr : (const T*)pv.data + h * pv.head + (int64_t)(j % a.pages.page) * pv.token + p * pv.page;
}

// ---------------------------------------------------------------- forward
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) fma_fwd_kernel(const __grid_constant__ SeqArgs a) {
    extern __shared__ float4 smem4[];
    constexpr int P = kPitch<DM>;
    float *Q = (float*)smem4, *K = Q + kTile * P, *V = K + kTile * P, *Pm = V + kTile * P;
    __shared__ unsigned char gone[kTile];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y;
    int tile = blockIdx.x;
    Seq s;
    if (a.pages.table) {
        if (!paged_seq(a, kTile, tile, &s)) return;
    } else {
        s = dense_seq(a, blockIdx.z);
    }
    const int rows = s.T * a.G, R0 = tile * kTile;
    const int p_lo = s.base + R0 / a.G, p_hi = s.base + (min(R0 + kTile, rows) - 1) / a.G;
    {
        const int r = tid >> 2, R = R0 + r, pos = s.base + R / a.G;
        load_row<T, DM>(Q + r * P, R < rows && pos >= 0 && pos < s.n ? row_ptr<T>(a.q, a, s, h, R) : nullptr, a.D, tid & 3);
    }
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, kTile);
    float m[4], l[4], o[4][DM / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DM / 16; ++c) o[i][c] = 0.f;
    }
    for (int it = 0; it < kt.count; ++it) {
        const int j0 = kt.key(it, kTile);
        __syncthreads();
        {
            const int r = tid >> 2, j = j0 + r;
            const T* kr = key_ptr<T>(a.k, a.kp, a, s, h, j);
            load_row<T, DM>(K + r * P, kr, a.D, tid & 3);
            // rows of v that no query of this tile sees may hold anything: they count as zeros
            const bool used = kr && (j >= p_lo - a.left || j < a.sinks) && j <= (int64_t)p_hi + a.right;
            load_row<T, DM>(V + r * P, used ? key_ptr<T>(a.v, a.vp, a, s, h, j) : nullptr, a.D, tid & 3);
            if (!(tid & 3)) gone[r] = !kr;
        }
        __syncthreads();
        float sc[4][4];
        dot_tile<DM>(Q, K, ty, tx, sc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int R = R0 + ty + 16 * i, pos = s.base + R / a.G;
            float top = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool see = R < rows && sees(a, s.n, pos, j0 + tx + 16 * j) && !gone[tx + 16 * j];
                sc[i][j] = see ? sc[i][j] * a.scale_log2 : -INFINITY;
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
#pragma unroll
            for (int c = 0; c < DM / 16; ++c) o[i][c] *= f;
        }
        __syncwarp();                                             // rows ty + 16i are written and read by one half warp
        acc_tile<DM>(Pm, V, ty, tx, o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int R = R0 + ty + 16 * i;
        if (R >= rows) continue;
        const float sum = sum16(l[i]);
        store_row<T, DM>(row_ptr<T>(a.y, a, s, h, R), o[i], sum > 0.f ? 1.f / sum : 0.f, a.D, tx);
        if (sizeof(T) == 2 && a.rest.data) {
            const float f = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
            for (int c = 0; c < DM / 16; ++c) o[i][c] = o[i][c] * f - to_float(from_float<T>(o[i][c] * f));
            store_row<T, DM>(row_ptr<T>(a.rest, a, s, h, R), o[i], 1.f, a.D, tx);
        }
        if (a.lse && tx == 0) a.lse[((int64_t)s.b * a.Hkv + h) * rows + R] = sum > 0.f ? m[i] + log2f(sum) : -INFINITY;
    }
}

// ---------------------------------------------------------------- backward
// P = 2^(scale q.k log2 e - lse), dP = dy.v, dS = P (dP - delta), delta = dy.y; dq = scale dS k.
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) fma_dq_kernel(const __grid_constant__ SeqArgs a) {
    extern __shared__ float4 smem4[];
    constexpr int P = kPitch<DM>;
    float *Q = (float*)smem4, *O = Q + kTile * P, *K = O + kTile * P, *V = K + kTile * P, *Pm = V + kTile * P;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y;
    const Seq s = dense_seq(a, blockIdx.z);
    const int rows = s.T * a.G, R0 = blockIdx.x * kTile;
    const int p_lo = R0 / a.G, p_hi = (min(R0 + kTile, rows) - 1) / a.G;
    const int64_t stat0 = ((int64_t)s.b * a.Hkv + h) * rows;
    float *yrow = K, *rest = V;                                   // y passes through the keys' place
    {
        const int r = tid >> 2, R = R0 + r;
        const bool live = R < rows && R / a.G < s.n;
        load_row<T, DM>(Q + r * P, live ? row_ptr<T>(a.q, a, s, h, R) : nullptr, a.D, tid & 3);
        load_row<T, DM>(O + r * P, live ? row_ptr<T>(a.dy, a, s, h, R) : nullptr, a.D, tid & 3);
        load_row<T, DM>(yrow + r * P, live ? row_ptr<T>(a.y, a, s, h, R) : nullptr, a.D, tid & 3);
        load_row<T, DM>(rest + r * P, live && a.rest.data ? row_ptr<T>(a.rest, a, s, h, R) : nullptr, a.D, tid & 3);
    }
    __syncthreads();
    float lse[4], delta[4], o[4][DM / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i, R = R0 + r;
        float d = 0.f;
        for (int f = tx; f < DM; f += 16) d = fmaf(O[r * P + f], yrow[r * P + f] + rest[r * P + f], d);
        delta[i] = sum16(d);
        lse[i] = R < rows ? a.lse[stat0 + R] : -INFINITY;
        if (R < rows && tx == 0) a.delta[stat0 + R] = delta[i];
#pragma unroll
        for (int c = 0; c < DM / 16; ++c) o[i][c] = 0.f;
    }
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, kTile);
    for (int it = 0; it < kt.count; ++it) {
        const int j0 = kt.key(it, kTile);
        __syncthreads();
        {
            const int r = tid >> 2, j = j0 + r;
            load_row<T, DM>(K + r * P, key_ptr<T>(a.k, a.kp, a, s, h, j), a.D, tid & 3);
            load_row<T, DM>(V + r * P, key_ptr<T>(a.v, a.vp, a, s, h, j), a.D, tid & 3);
        }
        __syncthreads();
        float sc[4][4], dp[4][4];
        dot_tile<DM>(Q, K, ty, tx, sc);
        dot_tile<DM>(O, V, ty, tx, dp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int R = R0 + ty + 16 * i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool see = R < rows && sees(a, s.n, R / a.G, j0 + tx + 16 * j);
                const float p = see ? fast_exp2(sc[i][j] * a.scale_log2 - lse[i]) : 0.f;
                Pm[(ty + 16 * i) * kPPitch + tx + 16 * j] = see ? p * (dp[i][j] - delta[i]) : 0.f;
            }
        }
        __syncwarp();
        acc_tile<DM>(Pm, K, ty, tx, o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int R = R0 + ty + 16 * i;
        if (R < rows) store_row<T, DM>(row_ptr<T>(a.dq, a, s, h, R), o[i], a.scale, a.D, tx);
    }
}

// A block owns 64 keys and walks the query rows that see any of them: dv = P^T dy, dk = scale dS^T q, no atomics.
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) fma_dkdv_kernel(const __grid_constant__ SeqArgs a) {
    extern __shared__ float4 smem4[];
    constexpr int P = kPitch<DM>;
    float *K = (float*)smem4, *V = K + kTile * P, *Q = V + kTile * P, *O = Q + kTile * P, *Pm = O + kTile * P, *Sm = Pm + kTile * kPPitch;
    __shared__ float s_lse[kTile], s_delta[kTile];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, h = blockIdx.y, j0 = blockIdx.x * kTile;
    const Seq s = dense_seq(a, blockIdx.z);
    const int rows = s.T * a.G;
    const int64_t stat0 = ((int64_t)s.b * a.Hkv + h) * rows;
    {
        const int r = tid >> 2;
        load_row<T, DM>(K + r * P, key_ptr<T>(a.k, a.kp, a, s, h, j0 + r), a.D, tid & 3);
        load_row<T, DM>(V + r * P, key_ptr<T>(a.v, a.vp, a, s, h, j0 + r), a.D, tid & 3);
    }
    float dk[4][DM / 16], dv[4][DM / 16];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DM / 16; ++c) dk[i][c] = dv[i][c] = 0.f;
    const int t_lo = max(0, j0 - a.right);
    const int t_hi = j0 < a.sinks ? s.n : (int)min((int64_t)s.n, (int64_t)j0 + kTile + a.left);
    for (int R0 = t_lo * a.G; R0 < t_hi * a.G && j0 < s.n; R0 += kTile) {
        __syncthreads();
        {
            const int r = tid >> 2, R = R0 + r;
            const bool live = R < t_hi * a.G;
            load_row<T, DM>(Q + r * P, live ? row_ptr<T>(a.q, a, s, h, R) : nullptr, a.D, tid & 3);
            load_row<T, DM>(O + r * P, live ? row_ptr<T>(a.dy, a, s, h, R) : nullptr, a.D, tid & 3);
            if (tid < kTile) {
                const bool have = R0 + tid < t_hi * a.G;
                s_lse[tid] = have ? a.lse[stat0 + R0 + tid] : 0.f;
                s_delta[tid] = have ? a.delta[stat0 + R0 + tid] : 0.f;
            }
        }
        __syncthreads();
        float sc[4][4], dp[4][4];
        dot_tile<DM>(K, Q, ty, tx, sc);
        dot_tile<DM>(V, O, ty, tx, dp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + ty + 16 * i;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int R = R0 + tx + 16 * c;
                const bool see = R < t_hi * a.G && sees(a, s.n, R / a.G, j);
                const float p = see ? fast_exp2(sc[i][c] * a.scale_log2 - s_lse[tx + 16 * c]) : 0.f;
                Pm[(ty + 16 * i) * kPPitch + tx + 16 * c] = p;
                Sm[(ty + 16 * i) * kPPitch + tx + 16 * c] = see ? p * (dp[i][c] - s_delta[tx + 16 * c]) : 0.f;
            }
        }
        __syncwarp();
        acc_tile<DM>(Pm, O, ty, tx, dv);
        acc_tile<DM>(Sm, Q, ty, tx, dk);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = j0 + ty + 16 * i;
        if (j >= a.N) continue;
        store_row<T, DM>((T*)a.dk.data + h * a.dk.head + (int64_t)j * a.dk.token + s.b * a.dk.batch, dk[i], a.scale, a.D, tx);
        store_row<T, DM>((T*)a.dv.data + h * a.dv.head + (int64_t)j * a.dv.token + s.b * a.dv.batch, dv[i], 1.f, a.D, tx);
    }
}

template <typename K>
int raise_smem(K kernel, size_t bytes) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? CA_OK : cuda_fail(e, "cudaFuncSetAttribute");
}

template <typename T, int DM>
int launch_fwd(const SeqArgs& a, cudaStream_t st) {
    const size_t smem = (3 * kTile * kPitch<DM> + kTile * kPPitch) * sizeof(float);
    const int rc = raise_smem(fma_fwd_kernel<T, DM>, smem);
    if (rc) return rc;
    const int64_t tiles = a.pages.table ? paged_tiles(a.N, a.G, a.pages.sequences, kTile) : ((int64_t)a.N * a.G + kTile - 1) / kTile;
    const dim3 grid((unsigned)tiles, a.Hkv, a.B);
    fma_fwd_kernel<T, DM><<<grid, kThreads, smem, st>>>(a);
    CA_CHECK_LAUNCH("window forward kernel");
    return CA_OK;
}

template <typename T, int DM>
int launch_bwd(const SeqArgs& a, cudaStream_t st) {
    const size_t smem_q = (4 * kTile * kPitch<DM> + kTile * kPPitch) * sizeof(float), smem_k = smem_q + kTile * kPPitch * sizeof(float);
    int rc = raise_smem(fma_dq_kernel<T, DM>, smem_q);
    if (rc || (rc = raise_smem(fma_dkdv_kernel<T, DM>, smem_k))) return rc;
    fma_dq_kernel<T, DM><<<dim3((unsigned)(((int64_t)a.N * a.G + kTile - 1) / kTile), a.Hkv, a.B), kThreads, smem_q, st>>>(a);
    CA_CHECK_LAUNCH("window dq kernel");
    fma_dkdv_kernel<T, DM><<<dim3((a.N + kTile - 1) / kTile, a.Hkv, a.B), kThreads, smem_k, st>>>(a);
    CA_CHECK_LAUNCH("window dk/dv kernel");
    return CA_OK;
}

}  // namespace

#define CA_SEQ_DISPATCH(dtype, D, FN, ...)                                                                            \
    do {                                                                                                             \
        const bool wide = (D) > 64;                                                                                  \
        if ((dtype) == CA_F32) return wide ? FN<float, 128>(__VA_ARGS__) : FN<float, 64>(__VA_ARGS__);               \
        if ((dtype) == CA_BF16) return wide ? FN<__nv_bfloat16, 128>(__VA_ARGS__) : FN<__nv_bfloat16, 64>(__VA_ARGS__); \
        return wide ? FN<__half, 128>(__VA_ARGS__) : FN<__half, 64>(__VA_ARGS__);                                    \
    } while (0)

int fma_window_fwd(const SeqArgs& a, int dtype, cudaStream_t st) { CA_SEQ_DISPATCH(dtype, a.D, launch_fwd, a, st); }
int fma_window_bwd(const SeqArgs& a, int dtype, cudaStream_t st) { CA_SEQ_DISPATCH(dtype, a.D, launch_bwd, a, st); }
int fma_paged(const SeqArgs& a, int dtype, cudaStream_t st) { CA_SEQ_DISPATCH(dtype, a.D, launch_fwd, a, st); }

}  // namespace ca
