// tcgen05 matrix instructions, tensor memory and the barriers around them, for one CTA.
//
// Operands in shared memory are rows of 64 16-bit elements (128 bytes) in the 128-byte swizzle that TMA writes: 16-byte
// piece c of row r sits at piece c ^ (r % 8), eight rows make an atom of 1024 bytes.  A tile of `rows` rows and DM features
// is DM/64 such panels, one behind the other.  The same bytes serve as an operand whose contraction runs along the features
// (K-major: scores) or along the rows (MN-major: weighted sums).
#pragma once
#include "tma.cuh"

namespace ca {

// ---------------------------------------------------------------- descriptors
constexpr uint32_t kPanel = 128 * 128;          // bytes of a panel of 128 rows

// Start address, leading and stride byte offsets in units of 16 bytes, version 1, 128-byte swizzle.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// Features are contracted: sixteen of them are 32 bytes of a row; 8-row groups are 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_features(uint32_t addr) { return smem_desc(addr, 16, 1024); }
// Rows are contracted: sixteen of them are 2048 bytes; the next 64 features are a panel further.
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr) { return smem_desc(addr, kPanel, 1024); }

// Float32 accumulator, A and B both bfloat16 or both half, M = 128; `rows_b`: B is contracted along its rows.
__host__ __device__ constexpr uint32_t instr_desc(bool bf16, int N, bool rows_b) {
    return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (rows_b ? 1u << 16 : 0u) | (uint32_t)(N >> 3) << 17 | (128u >> 4) << 24;
}

// ---------------------------------------------------------------- instructions (a warp in step, one lane issues)
// The warp that issues products runs as a whole; `lead` is set in one elected lane and guards the instruction itself, not a
// branch: control flow stays uniform, and descriptors are computed in the uniform registers that the instruction reads.
// As a branch of one lane the same code took 56 to 104 cycles an instruction, more than the product itself (64).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(lead) : "memory");
}
// The barrier gets one arrival when everything that the lane has issued so far is complete.
__device__ __forceinline__ void mma_commit(uint32_t lead, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}

// Tile times tile: D[128, 128] = A[128 rows] . B[128 rows]^T over DM features; desc_features of both.
template <int DM>
__device__ __forceinline__ void mma_dot(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
    for (int k = 0; k < DM / 16; ++k)         // addresses stand in units of 16 bytes in a descriptor's lowest bits
        mma_ss(lead, d, a + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, b + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, idesc, k != 0);
}
// The same with the rows of A in tensor memory, as 16-bit pairs.
template <int DM>
__device__ __forceinline__ void mma_dot_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
    for (int k = 0; k < DM / 16; ++k) mma_ts(lead, d, a + k * 8, b + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, idesc, k != 0);
}
// D[128, N] (+)= A[128, KEYS] in tensor memory (16-bit pairs) . B[KEYS rows, N]; desc_rows of B.
template <int KEYS>
__device__ __forceinline__ void mma_weighted(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
#pragma unroll
    for (int k = 0; k < KEYS / 16; ++k) mma_ts(lead, d, a + k * 8, b + k * 128, idesc, add || k != 0);
}

// ---------------------------------------------------------------- tensor memory (whole warps)
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, uint32_t columns) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 consecutive columns of this warp's 32 lanes; thread = lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
          "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
          "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
          "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}

// ---------------------------------------------------------------- bounded waits of a CTA with several roles
// A wait that runs out raises the CTA's flag, and every other wait of the CTA gives up when it sees it.
// The loop stands outside the callers' code: inlined, a wait for a barrier that is long complete took 300 cycles, not 100.
static __device__ __noinline__ bool keep_waiting(uint32_t bar, uint32_t parity, volatile int* stop) {
    for (int i = 0; i < 64; ++i) {
        if (mbar_wait(bar, parity, 1u << 14)) return true;
        if (*stop) return false;
    }
    *stop = 1;
    return false;
}
__device__ __forceinline__ bool wait_or_stop(uint32_t bar, uint32_t parity, volatile int* stop) {
    return mbar_wait(bar, parity, 1) || keep_waiting(bar, parity, stop);
}
// The same for a whole warp, which then goes on or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* stop) {
    if (__all_sync(~0u, mbar_wait(bar, parity, 1))) return true;
    return __all_sync(~0u, keep_waiting(bar, parity, stop));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---------------------------------------------------------------- pairs of Float32
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// ---------------------------------------------------------------- host side
// Tensor map of 16-bit elements in the 128-byte swizzle; `dims` innermost first, `strides_bytes` for dims 1..rank-1.
int encode_swizzled_map(CUtensorMap* map, bool bf16, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes,
                        const uint32_t* box);
int* stage_timeout_counter();

}  // namespace ca
