// Attention on token sequences, forward: tensor maps and the choice of the kernel (seq_fwd.cuh), and the kernels of plain scores.
#include "seq_fwd.cuh"

namespace ca {

extern template int umma_fwd<kSlopes>(const SeqArgs&, const FwdMaps&, int, bool, dim3, cudaStream_t);
extern template int umma_fwd<kCap>(const SeqArgs&, const FwdMaps&, int, bool, dim3, cudaStream_t);
extern template int umma_fwd<kCapSlopes>(const SeqArgs&, const FwdMaps&, int, bool, dim3, cudaStream_t);

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

// bfloat16's exponents hold the weights of capped scores without a look for their maximum, and Float32's what they multiply, up to a
// cap of 33 (kOnePassCap).  Half's do not, and larger caps leave no room for the values: those take the kernel that looks (16384 tokens,
// window 1024, 16 and 4 heads of 128 features, scores of standard deviation 8: 266 us with one pass, 345 with two; cap 30, a few scores
// beyond the cap, 292 and 354).
static int run(const SeqArgs& a, const FwdMaps& maps, int dtype, bool pair, dim3 grid, cudaStream_t st) {
    switch (a.kind) {
        case kMasks: return umma_fwd<kMasks>(a, maps, dtype, pair, grid, st);
        case kSlopes: return umma_fwd<kSlopes>(a, maps, dtype, pair, grid, st);
        case kCap:
            if (dtype == CA_BF16 && a.form.cap_out <= kOnePassCap) return umma_fwd<kCap>(a, maps, dtype, pair, grid, st);
            [[fallthrough]];
        case kCapSlopes: return umma_fwd<kCapSlopes>(a, maps, dtype, pair, grid, st);
        default: return umma_fwd<kNoForm>(a, maps, dtype, pair, grid, st);
    }
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
    const dim3 grid((unsigned)((rows + (pair ? 255 : 127)) / (pair ? 256 : 128)), a.Hkv, a.B);
    maps.ranked = a.form.spans && (int64_t)grid.x * grid.y * grid.z > sm_count();             // else all blocks start at once
    return run(a, maps, dtype, pair, grid, st);
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
    const dim3 grid((unsigned)tiles, a.Hkv, 1);
    return run(a, maps, dtype, pair, grid, st);
}

}  // namespace ca
