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

// The registers of a tensor-memory load are complete behind its wait: nothing that uses them may move before it.
__device__ __forceinline__ void settled32(uint32_t* r) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// One row of D elements into a swizzled tile of DM features, zeros behind D and where `src` is null; pieces from `first` on,
// every `step`-th.  `flip`: the sign is turned.
template <typename T, int DM>
__device__ __forceinline__ void stage_row(char* tile, int r, const T* src, int D, int first, int step, bool flip) {
    const uint32_t sign = flip ? 0x80008000u : 0u;
#pragma unroll 8
    for (int c = first; c < DM / 8; c += step) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (src && c * 8 < D) w = *reinterpret_cast<const uint4*>(src + c * 8);
        w.x ^= sign; w.y ^= sign; w.z ^= sign; w.w ^= sign;
        *reinterpret_cast<uint4*>(tile + (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
    }
}

// Bits 0..31 of the columns c with lo <= c <= hi or c < sk, c <= hi.
__device__ __forceinline__ uint32_t bits_upto(int h) { return h < 0 ? 0u : h >= 31 ? ~0u : (2u << h) - 1u; }
__device__ __forceinline__ uint32_t bits_from(int l) { return l <= 0 ? ~0u : l > 31 ? 0u : ~0u << l; }
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int sk) { return bits_upto(hi) & (bits_from(lo) | bits_upto(sk - 1)); }

template <typename T>
__device__ __forceinline__ T* seq_row(const ca_seq_view& v, const SeqArgs& a, const Seq& s, int h, int R) {
    const int t = R / a.G, g = R - t * a.G;
    return (T*)v.data + (h * a.G + g) * v.head + (int64_t)(s.t0 + t) * v.token + (a.pages.table ? 0 : s.b * v.batch);
}

// Counts a CTA that gave up a wait and flags it for the host.
__device__ __forceinline__ void report_stop(int* timeouts, int* status) {
    atomicAdd(timeouts, 1);
    if (status) atomicOr(status, 1);
}

// Dense keys (D, tokens, heads, batch), boxes of 64 features and 128 tokens.
int encode_tokens(CUtensorMap* m, bool bf16, const ca_seq_view& v, int D, int heads, int tokens, int batch, int box_tokens);

// seq_fwd.cu
int umma_window_fwd(const SeqArgs& a, int dtype, cudaStream_t st);
int umma_paged(const SeqArgs& a, int dtype, cudaStream_t st);
// seq_bwd.cu
size_t umma_bwd_parts(const SeqArgs& a);
int umma_window_bwd(const SeqArgs& a, int dtype, float* parts, cudaStream_t st);

}  // namespace ca
