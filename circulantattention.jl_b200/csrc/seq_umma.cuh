// Parts that the tensor-core kernels of the attention on token sequences share.
#pragma once
#include "seq.cuh"
#include "umma.cuh"

namespace ca {

template <typename T> constexpr bool kIsBf16 = sizeof(T) == 2;      // specialised below
template <> constexpr bool kIsBf16<__half> = false;

// Two Float32 -> two 16-bit elements, `lo` in the lower half.
template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ float low16(uint32_t w) { return to_float(reinterpret_cast<const T*>(&w)[0]); }
template <typename T> __device__ __forceinline__ float high16(uint32_t w) { return to_float(reinterpret_cast<const T*>(&w)[1]); }

// The larger of two numbers; not a number if one of them is not
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x for two numbers below 2^7 on the FMA pipe: x = n + f with n the nearest integer (the low bits of x + 1.5 2^23), a
// polynomial for 2^f on [-1/2, 1/2], times 2^n; 0 below 2^-126.  The coefficients minimise the largest relative error (Lawson's
// iteration): 7.5e-5 with degree 3, below the rounding to bfloat16 that follows by a factor of 26; 2.6e-6 with degree 4 for
// half.  A number that is not one stays so, as in the other exponentials.
template <typename T>
__device__ __forceinline__ f32x2 exp2_fma(float x0, float x1) {
    const f32x2 magic = pack2(12582912.f, 12582912.f), unmagic = pack2(-12582912.f, -12582912.f), minus = pack2(-1.f, -1.f);
    const f32x2 x = pack2(max_nan(x0, -127.f), max_nan(x1, -127.f));
    const f32x2 t = add2(x, magic);
    const f32x2 f = fma2(add2(t, unmagic), minus, x);
    f32x2 p;
    if (kIsBf16<T>) {
        p = fma2(f, pack2(0.055171494f, 0.055171494f), pack2(0.242610938f, 0.242610938f));
        p = fma2(f, p, pack2(0.693260994f, 0.693260994f));
        p = fma2(f, p, pack2(0.999928085f, 0.999928085f));
    } else {
        p = fma2(f, pack2(0.00957008612f, 0.00957008612f), pack2(0.055917851f, 0.055917851f));
        p = fma2(f, p, pack2(0.240247451f, 0.240247451f));
        p = fma2(f, p, pack2(0.693121816f, 0.693121816f));
        p = fma2(f, p, pack2(0.999999261f, 0.999999261f));
    }
    float t0, t1;
    unpack2(t, t0, t1);
    return mul2(p, pack2(__uint_as_float((__float_as_uint(t0) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(t1) << 23) + 0x3f800000u)));
}

// The registers of a tensor-memory load are complete behind its wait: nothing that uses them may move before it.
__device__ __forceinline__ void settled32(uint32_t* r) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// Tiles between global and shared memory: consecutive threads take consecutive 16-byte pieces of a row, so that a warp covers
// two to four whole rows at a time (a thread for each row would touch 32 lines an instruction: 4096 cycles a tile of 128 rows,
// and three such tiles made the prologue of dq 10 us).  `row(r)`: address of row r.  Rows
// from..to-1 exist; others are zeros, or not stored.  Addresses are computed without branches, so that they overlap.
template <int DM, int THREADS> struct TileCopy {
    static constexpr int kPieces = DM / 8, kStep = THREADS / kPieces, kCount = 128 / kStep;
    static __device__ __forceinline__ int piece(int tid) { return tid % kPieces; }
    static __device__ __forceinline__ int row(int tid, int i) { return tid / kPieces + i * kStep; }
    static __device__ __forceinline__ uint32_t at(int r, int c) { return (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
};

template <typename T, int DM, int THREADS, typename Row>
__device__ __forceinline__ void fetch_tile(uint4 (&w)[TileCopy<DM, THREADS>::kCount], Row row, int from, int to, int D, int tid) {
    typedef TileCopy<DM, THREADS> C;
    const int c = C::piece(tid);
#pragma unroll
    for (int i = 0; i < C::kCount; ++i) {
        const int r = C::row(tid, i);
        const T* src = row(min(max(r, from), max(to - 1, from)));
        w[i] = make_uint4(0, 0, 0, 0);
        if (r >= from && r < to && c * 8 < D) w[i] = *reinterpret_cast<const uint4*>(src + c * 8);
    }
}
template <int DM, int THREADS>
__device__ __forceinline__ void put_tile(char* tile, const uint4 (&w)[TileCopy<DM, THREADS>::kCount], int tid) {
    typedef TileCopy<DM, THREADS> C;
#pragma unroll
    for (int i = 0; i < C::kCount; ++i) *reinterpret_cast<uint4*>(tile + C::at(C::row(tid, i), C::piece(tid))) = w[i];
}
template <typename T, int DM, int THREADS, typename Row>
__device__ __forceinline__ void store_tile(const char* tile, Row row, int to, int D, int tid) {
    typedef TileCopy<DM, THREADS> C;
    const int c = C::piece(tid);
    uint4 w[C::kCount];
#pragma unroll
    for (int i = 0; i < C::kCount; ++i) w[i] = *reinterpret_cast<const uint4*>(tile + C::at(C::row(tid, i), c));
#pragma unroll
    for (int i = 0; i < C::kCount; ++i) {
        const int r = C::row(tid, i);
        T* dst = row(min(r, to - 1));
        if (r < to && c * 8 < D) *reinterpret_cast<uint4*>(dst + c * 8) = w[i];
    }
}
// 32 results of row r, columns first .. first + 31, into a tile that store_tile takes.
template <typename T>
__device__ __forceinline__ void put_row32(char* tile, int r, int first, const float* y) {
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
        const int c = (first + e) >> 3;
        *reinterpret_cast<uint4*>(tile + (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
            make_uint4(pack16<T>(y[e], y[e + 1]), pack16<T>(y[e + 2], y[e + 3]), pack16<T>(y[e + 4], y[e + 5]), pack16<T>(y[e + 6], y[e + 7]));
    }
}
// All threads of one or two warpgroups (named barrier `id`); every one of them gets here on every path.
template <int THREADS> __device__ __forceinline__ void group_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory"); }

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }

// Bits 0..31 of the columns c with lo <= c <= hi or c < sk, c <= hi.
__device__ __forceinline__ uint32_t bits_upto(int h) { return h < 0 ? 0u : h >= 31 ? ~0u : (2u << h) - 1u; }
__device__ __forceinline__ uint32_t bits_from(int l) { return l <= 0 ? ~0u : l > 31 ? 0u : ~0u << l; }
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int sk) { return bits_upto(hi) & (bits_from(lo) | bits_upto(sk - 1)); }

template <typename T>
__device__ __forceinline__ T* seq_row(const ca_seq_view& v, const SeqArgs& a, const Seq& s, int h, int R) {
    const int t = token_of(a, R), g = R - t * a.G;
    return (T*)v.data + (h * a.G + g) * v.head + (int64_t)(s.t0 + t) * v.token + (a.pages.table ? 0 : s.b * v.batch);
}

// Counts a CTA that gave up a wait and flags it for the host.
__device__ __forceinline__ void report_stop(int* timeouts, int* status) {
    atomicAdd(timeouts, 1);
    if (status) atomicOr(status, 1);
}

// One head's tokens, (D, tokens, heads, batch): boxes of 64 features and 128 tokens, coordinates (feature, token, head, batch).
int encode_tokens(CUtensorMap* m, bool bf16, const ca_seq_view& v, int D, int heads, int tokens, int batch);
// Tiles of 128 packed rows, (D, heads, tokens, batch): boxes of 64 features, the G heads of a group and 128 / G tokens.
// G divides 128 (rows_fit); with other groups rows are copied by threads.
static inline bool rows_fit(const SeqArgs& a) { return 128 % a.G == 0; }
int encode_rows(CUtensorMap* m, bool bf16, const ca_seq_view& v, const SeqArgs& a);

// Stores a tile (as put_row32 leaves it) through a map; one thread, after fence_async_smem and a barrier of the writers.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// Brings a box into L2.
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];"
                 ::"l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// The stores of this thread have read their shared memory.
__device__ __forceinline__ void tma_stores_read() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// seq_fwd.cu
int umma_window_fwd(const SeqArgs& a, int dtype, cudaStream_t st);
int umma_paged(const SeqArgs& a, int dtype, cudaStream_t st);
// seq_decode.cu: few rows a key head, every type
int decode_paged(const SeqArgs& a, int dtype, cudaStream_t st);
// seq_bwd.cu
size_t umma_bwd_parts(const SeqArgs& a);
int umma_window_bwd(const SeqArgs& a, int dtype, float* parts, cudaStream_t st);

}  // namespace ca
