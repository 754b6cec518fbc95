// What each token sees and which tokens see it, from the numbers of documents and groups.
//
// A run (document or group) begins at a token whose number differs from the one before, so the begin of a token's run is the
// largest such place up to it, and its end lies before the smallest one behind it: two scans.  A cluster takes a sequence, a
// thread a piece of consecutive tokens: it finds the first and the last place in its piece, places are joined over warps,
// the block and the cluster, and then it walks its piece again, forwards for the begins and backwards for the ends.
//
// Bound: latency.  300 tokens 2.6 us, 16384 in a cluster of eight blocks 7.6 us (9.8 with the warps' and blocks' places read one by
// one).
#include <cooperative_groups.h>
#include <limits.h>
#include "seq.cuh"

namespace cg = cooperative_groups;

namespace ca {
namespace {

constexpr int kSpanThreads = 1024, kSpanWarps = kSpanThreads / 32;

struct SpanArgs {
    const int *documents, *groups;      // [batch][token]; groups nullable
    int* spans;                         // [batch][token][4]
    int N;
};

// Places where documents and groups begin: the last ones so far, or the first ones from here on.
struct Places { int document, group; };
__device__ __forceinline__ Places later(Places a, Places b) { return Places{max(a.document, b.document), max(a.group, b.group)}; }
__device__ __forceinline__ Places sooner(Places a, Places b) { return Places{min(a.document, b.document), min(a.group, b.group)}; }

__global__ void __launch_bounds__(kSpanThreads) span_kernel(const __grid_constant__ SpanArgs a) {
    __shared__ Places warp_last[kSpanWarps], warp_first[kSpanWarps], block_last, block_first;
    let_next_begin();
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y;
    const int* documents = a.documents + (int64_t)b * a.N;
    const int* groups = a.groups ? a.groups + (int64_t)b * a.N : nullptr;
    int* spans = a.spans + (int64_t)b * a.N * 4;
    const int piece = (a.N + ranks * kSpanThreads - 1) / (ranks * kSpanThreads);
    const int64_t at = (int64_t)piece * (rank * kSpanThreads + tid);
    const int from = (int)min((int64_t)a.N, at), to = (int)min((int64_t)a.N, at + piece);
    auto group_of = [&](int i) { return groups ? groups[i] : 0; };

    Places last{-1, -1}, first{a.N, a.N};
    if (from < to) {
        int d = from ? documents[from - 1] : 0, g = from ? group_of(from - 1) : 0;
        for (int i = from; i < to; ++i) {
            const int dn = documents[i], gn = group_of(i);
            const bool nd = i == 0 || dn != d, ng = nd || gn != g;
            if (nd) last.document = i, first.document = min(first.document, i);
            if (ng) last.group = i, first.group = min(first.group, i);
            d = dn;
            g = gn;
        }
    }
    // places before this thread's piece, and behind it
    Places before = last, behind = first;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Places x{__shfl_up_sync(~0u, before.document, o), __shfl_up_sync(~0u, before.group, o)};
        const Places y{__shfl_down_sync(~0u, behind.document, o), __shfl_down_sync(~0u, behind.group, o)};
        if (lane >= o) before = later(before, x);
        if (lane + o < 32) behind = sooner(behind, y);
    }
    if (lane == 31) warp_last[warp] = before;
    if (lane == 0) warp_first[warp] = behind;
    before = Places{__shfl_up_sync(~0u, before.document, 1), __shfl_up_sync(~0u, before.group, 1)};
    behind = Places{__shfl_down_sync(~0u, behind.document, 1), __shfl_down_sync(~0u, behind.group, 1)};
    if (lane == 0) before = Places{-1, -1};
    if (lane == 31) behind = Places{a.N, a.N};
    __syncthreads();
    // every warp joins the warps' places, a lane for each, and then the blocks'
    auto join = [&](Places last, Places first, int own) {
        before = later(before, Places{__reduce_max_sync(~0u, lane < own ? last.document : -1), __reduce_max_sync(~0u, lane < own ? last.group : -1)});
        behind = sooner(behind, Places{__reduce_min_sync(~0u, lane > own ? first.document : a.N), __reduce_min_sync(~0u, lane > own ? first.group : a.N)});
    };
    const Places lasts = warp_last[lane], firsts = warp_first[lane];
    join(lasts, firsts, warp);
    if (ranks > 1) {
        if (warp == 0) {
            const Places all_last{__reduce_max_sync(~0u, lasts.document), __reduce_max_sync(~0u, lasts.group)};
            const Places all_first{__reduce_min_sync(~0u, firsts.document), __reduce_min_sync(~0u, firsts.group)};
            if (lane == 0) {
                block_last = all_last;
                block_first = all_first;
            }
        }
        cluster.sync();
        Places last{-1, -1}, first{a.N, a.N};
        if (lane < ranks) {
            last = *cluster.map_shared_rank(&block_last, lane);
            first = *cluster.map_shared_rank(&block_first, lane);
        }
        join(last, first, rank);
        cluster.sync();                                         // nobody leaves while its places are read
    }
    if (from >= to) return;
    {
        int d = from ? documents[from - 1] : 0, g = from ? group_of(from - 1) : 0;
        for (int i = from; i < to; ++i) {
            const int dn = documents[i], gn = group_of(i);
            const bool nd = i == 0 || dn != d, ng = nd || gn != g;
            if (nd) before.document = i;
            if (ng) before.group = i;
            *reinterpret_cast<int2*>(spans + (int64_t)i * 4) = dn < 0 ? make_int2(i, i) : make_int2(before.document, gn > 0 ? before.group : i);
            d = dn;
            g = gn;
        }
    }
    int d = documents[to - 1], g = group_of(to - 1);
    for (int i = to - 1; i >= from; --i) {
        *reinterpret_cast<int2*>(spans + (int64_t)i * 4 + 2) = d < 0 ? make_int2(i - 1, i - 1) : make_int2(g > 0 ? behind.group - 1 : i, behind.document - 1);
        if (i == 0) break;
        const int dp = documents[i - 1], gp = group_of(i - 1);
        if (dp != d) behind.document = i;
        if (dp != d || gp != g) behind.group = i;
        d = dp;
        g = gp;
    }
}

}  // namespace
}  // namespace ca

using namespace ca;

extern "C" int ca_token_spans(const int32_t* documents, const int32_t* groups, int32_t tokens, int32_t batch, int32_t* spans, void* stream) {
    if (tokens < 0 || batch < 0) { set_error("tokens=%d batch=%d must not be negative", tokens, batch); return CA_ERR_BAD_DESC; }
    if (tokens > kNoLeft || batch > 65535) { set_error("tokens=%d batch=%d exceed 2^30 tokens or the grid limit 65535", tokens, batch); return CA_ERR_TOO_LARGE; }
    if (!tokens || !batch) return CA_OK;
    if (!documents || !spans) { set_error("documents and spans must not be NULL"); return CA_ERR_NULL; }
    if (reinterpret_cast<uintptr_t>(spans) % 16 || reinterpret_cast<uintptr_t>(documents) % 4 || reinterpret_cast<uintptr_t>(groups) % 4) {
        set_error("documents, groups or spans (16 bytes) are not aligned");
        return CA_ERR_BAD_DESC;
    }
    // Up to eight blocks a sequence, as long as each thread has a token
    int ranks = 1;
    while (ranks < 8 && (int64_t)tokens > (int64_t)ranks * kSpanThreads) ranks *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(ranks, batch); cfg.blockDim = dim3(kSpanThreads); cfg.stream = as_stream(stream);
    cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, span_kernel, SpanArgs{documents, groups, spans, tokens});
    if (e != cudaSuccess) return cuda_fail(e, "span kernel");
    CA_CHECK_LAUNCH("span kernel");
    return CA_OK;
}
