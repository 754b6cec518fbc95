// The pages of a cache: taken and freed (a serving step), forked, compacted.
//
// The state is a table of pages for each sequence and, for each page, the number of table entries that hold it.  Each operator
// takes a state and gives the next one; where pages have to be copied it lists them, and a second kernel copies them in all
// pools.  Which page goes where is fixed by order, lowest numbers first, never by which thread comes first: the only atomics add
// and subtract whole numbers.
//
// The bookkeeping is a handful of passes over the table and the counts with a barrier between them.  One cluster of blocks does all
// of it in one launch: a cluster's barrier costs less than a launch, and its scans pass totals through distributed shared
// memory.  Bound: latency of the passes, and for the copies memory.
//
// Measured, bookkeeping and copies: a step of 64 sequences of 1880 places 13.6 us, of 256 with chunks (85000 pages) 19.5; a fork of 8 beams
// 8.3 + 3.3, of 128 samples (0.5 GB moved) 12.9 + 80 (the copies begin under the bookkeeping; floor 77); compaction of 300 pages 5.4 +
// 2.8, of 2000 (1.05 GB) 10 + 175 us, 6.0 TB/s.
#include <cooperative_groups.h>
#include <algorithm>
#include "seq.cuh"

namespace cg = cooperative_groups;

namespace ca {
namespace {

constexpr int kThreads = 1024, kBlocks = 16, kMovePools = 32;

struct PageArgs {
    ca_table t;
    const int *starts, *parents;
    int left, sinks;
    int *table, *refs, *lengths, *result;       // the next state; result: pages that were wanting, or pages in use
    int *list, *source, *target, *keeper, *need, *offset, *moves;      // offset: for each block
};

struct Team {
    cg::cluster_group cluster;
    int thread, threads, rank, ranks;
    __device__ __forceinline__ Team() : cluster(cg::this_cluster()), rank((int)cluster.block_rank()), ranks((int)cluster.num_blocks()) {
        thread = rank * kThreads + threadIdx.x;
        threads = ranks * kThreads;
    }
    // Everything that the cluster's threads wrote before is seen behind this (by loads that pass by the L1 cache)
    __device__ __forceinline__ void sync() const { cluster.sync(); }
    // Sum of v over the block's threads before this one, and over all of them
    __device__ int2 block_scan(int v) const {
        __shared__ int warps[kThreads / 32];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        int upto = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += x;
        }
        __syncthreads();                                        // the sums of a scan before have been read
        if (lane == 31) warps[warp] = upto;
        __syncthreads();
        int sum = warps[lane];                               // every warp scans the warps' sums
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += x;
        }
        const int before = __shfl_sync(~0u, sum, max(warp - 1, 0));
        return make_int2((warp ? before : 0) + upto - v, __shfl_sync(~0u, sum, 31));
    }
    // The same over the cluster.  SLOT: one for each scan of a kernel, so that no barrier has to guard the totals; a kernel's last
    // scan is followed by a barrier.
    template <int SLOT>
    __device__ int2 scan(int v) const {
        __shared__ int total[2];
        const int2 own = block_scan(v);
        if (ranks == 1) return own;
        if (threadIdx.x == 0) total[SLOT] = own.y;
        cluster.sync();
        const int lane = threadIdx.x & 31, x = lane < ranks ? *cluster.map_shared_rank(&total[SLOT], lane) : 0;      // a lane for each block
        return make_int2(own.x + __reduce_add_sync(~0u, lane < rank ? x : 0), __reduce_add_sync(~0u, x));
    }
};

// This thread's share of n consecutive things
__device__ __forceinline__ int2 share(const Team& team, int n) {
    const int piece = (n + team.threads - 1) / team.threads;
    const int64_t at = (int64_t)piece * team.thread;
    return make_int2((int)min((int64_t)n, at), (int)min((int64_t)n, at + piece));
}

__device__ __forceinline__ bool is_page(const ca_table& t, int e) { return e >= 0 && e < t.pages; }

// The places of the table, a warp for 128 places of one sequence: body(sequence, whatever of(sequence) is, place, index in the table).
constexpr int kPlaces = 128;
template <typename Of, typename Body>
__device__ __forceinline__ void for_places(const PageArgs& a, const Team& team, Of of, Body body) {
    const int W = a.t.width, pieces = (W + kPlaces - 1) / kPlaces, lane = threadIdx.x & 31;
    const int64_t units = (int64_t)pieces * a.t.sequences;
    for (int64_t unit = team.thread >> 5; unit < units; unit += team.threads >> 5) {
        const int s = units <= INT32_MAX ? (int)((uint32_t)unit / (uint32_t)pieces) : (int)(unit / pieces), c0 = (int)(unit - (int64_t)s * pieces) * kPlaces + lane;
        const auto x = of(s);
        int e[kPlaces / 32];
#pragma unroll
        for (int k = 0; k < kPlaces / 32; ++k) e[k] = c0 + 32 * k < W ? a.t.table[(int64_t)s * W + c0 + 32 * k] : -1;
#pragma unroll
        for (int k = 0; k < kPlaces / 32; ++k)
            if (c0 + 32 * k < W) body(s, x, c0 + 32 * k, (int64_t)s * W + c0 + 32 * k, e[k]);
    }
}

// The warp's share of the pages: whole groups of 32, so that its loads are of neighbours.
__device__ __forceinline__ int2 warp_pages(const PageArgs& a, const Team& team) {
    const int warps = team.threads >> 5, groups = (a.t.pages + 31) / 32, piece = (groups + warps - 1) / warps * 32;
    const int64_t at = (int64_t)piece * (team.thread >> 5);
    return make_int2((int)min((int64_t)a.t.pages, at), (int)min((int64_t)a.t.pages, at + piece));
}
// How many of the warp's pages are `picked`; known to its first lane, which stands for the warp in a scan.
template <typename Picked>
__device__ __forceinline__ int count_pages(int2 mine, Picked picked) {
    const int lane = threadIdx.x & 31;
    int count = 0;
#pragma unroll 4
    for (int i = mine.x + lane; i < mine.y; i += 32) count += picked(i);
    count = __reduce_add_sync(~0u, count);
    return lane == 0 ? count : 0;
}
// body(page, picked or not, pages picked before it) for the warp's pages, of which `before` come earlier; the warp in step.
template <typename Picked, typename Body>
__device__ __forceinline__ void number_pages(int2 mine, int before, Picked picked, Body body) {
    const int lane = threadIdx.x & 31;
    before = __shfl_sync(~0u, before, 0);
    for (int i0 = mine.x; i0 < mine.y; i0 += 32) {
        const int i = i0 + lane;
        const bool on = i < mine.y && picked(i);
        const unsigned all = __ballot_sync(~0u, on);
        if (i < mine.y) body(i, on, before + __popc(all & ((1u << lane) - 1)));
        before += __popc(all);
    }
}

// Lists the lowest `wanted` pages without users; returns how many of them there are.
__device__ int list_free(const PageArgs& a, const Team& team, int wanted) {
    const int2 mine = warp_pages(a, team);
    auto free = [&](int i) { return __ldcg(a.refs + i) <= 0; };
    const int2 rank = team.scan<0>(count_pages(mine, free));
    number_pages(mine, rank.x, free, [&](int i, bool on, int at) {
        if (on && at < wanted) a.list[at] = i;
    });
    return min(rank.y, wanted);
}

// Sums over the sequences before each, in place; every block does it for itself and returns the sum of all.
__device__ int offsets(const PageArgs& a, const Team& team, int* offset) {
    const int S = a.t.sequences, piece = (S + kThreads - 1) / kThreads;
    const int from = min(S, piece * (int)threadIdx.x), to = min(S, from + piece);
    int count = 0;
    for (int s = from; s < to; ++s) count += __ldcg(a.need + s);
    int2 rank = team.block_scan(count);
    for (int s = from; s < to; ++s) {
        offset[s] = rank.x;                                     // alike in all blocks
        rank.x += __ldcg(a.need + s);
    }
    return rank.y;
}

// ---------------------------------------------------------------- a serving step
// What stays of sequence s: the places first..upto - 1 and those below `sinks`; new tokens are in fresh..upto - 1.
struct Stay {
    int first, upto, sinks, fresh;
    __device__ __forceinline__ Stay(const PageArgs& a, int s) {
        const uint32_t page = a.t.page, n = max(0, a.t.lengths[s]);
        const int64_t count = (int64_t)a.starts[s + 1] - a.starts[s];
        const uint32_t begin = (uint32_t)max((int64_t)0, n - max((int64_t)0, count));
        upto = (int)min((uint32_t)a.t.width, (n + page - 1) / page);
        first = a.left < 0 ? 0 : (int)(begin > (uint32_t)a.left ? (begin - a.left) / page : 0);
        sinks = (int)((min((uint32_t)a.sinks, n) + page - 1) / page);
        fresh = count > 0 ? min(upto, (int)(begin / page)) : upto;
    }
    __device__ __forceinline__ bool has(int c) const { return c < upto && (c >= first || c < sinks); }
};

__global__ void __launch_bounds__(kThreads) advance_kernel(const __grid_constant__ PageArgs a) {
    const Team team;
    const int S = a.t.sequences, W = a.t.width, lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.t.pages; i += team.threads) a.refs[i] = a.t.refs[i];
    // a warp for each sequence: its new places without a page
    for (int s = team.thread >> 5; s < S; s += team.threads >> 5) {
        const Stay stay(a, s);
        int need = 0;
        for (int c = stay.fresh + lane; c < stay.upto; c += 32) need += !is_page(a.t, a.t.table[(int64_t)s * W + c]);
        need = __reduce_add_sync(~0u, need);
        if (lane == 0) a.need[s] = need;
    }
    team.sync();
    for_places(a, team, [&](int s) { return Stay(a, s); }, [&](int, const Stay& stay, int c, int64_t i, int e) {
        const bool there = is_page(a.t, e), stays = stay.has(c);
        if (there || c < stay.fresh || c >= stay.upto) a.table[i] = there && stays ? e : -1;       // other places get theirs below
        if (there && !stays) atomicSub(a.refs + e, 1);
    });
    int* const offset = a.offset + (size_t)team.rank * S;
    const int wanted = offsets(a, team, offset);
    team.sync();
    const int got = list_free(a, team, wanted);
    team.sync();
    for (int s = team.thread >> 5; s < S; s += team.threads >> 5) {
        const Stay stay(a, s);
        int at = offset[s];
        for (int c0 = stay.fresh; c0 < stay.upto; c0 += 32) {
            const int c = c0 + lane;
            const bool need = c < stay.upto && !is_page(a.t, a.t.table[(int64_t)s * W + c]);
            const unsigned all = __ballot_sync(~0u, need);
            const int k = at + __popc(all & ((1u << lane) - 1));
            if (need) {
                const int p = k < got ? __ldcg(a.list + k) : -1;
                a.table[(int64_t)s * W + c] = p;
                if (p >= 0) a.refs[p] = 1;
            }
            at += __popc(all);
        }
    }
    if (team.thread == 0) *a.result = wanted - got;
}

// ---------------------------------------------------------------- forking
__device__ __forceinline__ int parent_of(const PageArgs& a, int s) {
    const int p = a.parents[s];
    return p >= 0 && p < a.t.sequences ? p : -1;
}
// What sequence s becomes.
struct Child {
    int parent, full;           // places below `full` are the parent's
    bool part, keeps;           // the next one is partly filled; s keeps its page
    __device__ __forceinline__ Child(const PageArgs& a, int s) : parent(parent_of(a, s)) {
        const uint32_t n = parent < 0 ? 0u : (uint32_t)min((int64_t)max(0, a.t.lengths[parent]), (int64_t)a.t.width * a.t.page);
        full = n / (uint32_t)a.t.page;
        part = n % (uint32_t)a.t.page != 0;
        keeps = parent >= 0 && __ldcg(a.keeper + parent) == s;
    }
    // Whether it needs a copy of that page.
    __device__ __forceinline__ bool copies(const PageArgs& a, int s) const {
        return part && !keeps && parent != s && is_page(a.t, a.t.table[(int64_t)parent * a.t.width + full]);
    }
};

__global__ void __launch_bounds__(kThreads) fork_kernel(const __grid_constant__ PageArgs a) {
    const Team team;
    let_next_begin();
    const int S = a.t.sequences, W = a.t.width;
    for (int i = team.thread; i < a.t.pages; i += team.threads) a.refs[i] = a.t.refs[i];
    // the partly filled page stays with the parent if it goes on, else with the first sequence that continues it
    for (int s = team.thread; s < S; s += team.threads) {
        const int p = parent_of(a, s);
        a.lengths[s] = p < 0 ? 0 : a.t.lengths[p];
        a.keeper[s] = parent_of(a, s) == s ? -1 : S;
    }
    team.sync();
    for (int s = team.thread; s < S; s += team.threads) {
        const int p = parent_of(a, s);
        if (p >= 0 && p != s) atomicMin(a.keeper + p, s);
    }
    team.sync();
    for_places(a, team, [&](int s) { return Child(a, s); }, [&](int s, const Child& x, int c, int64_t i, int old) {
        int e = old;
        if (x.parent != s) {
            if (is_page(a.t, old)) atomicSub(a.refs + old, 1);
            e = -1;
            if (x.parent >= 0 && (c < x.full || (c == x.full && x.part && x.keeps))) {
                e = a.t.table[(int64_t)x.parent * W + c];
                if (is_page(a.t, e)) atomicAdd(a.refs + e, 1);
                else e = -1;
            }
        }
        if (c != x.full || !x.copies(a, s)) a.table[i] = e;     // copies get their page below
    });
    const int2 mine = share(team, S);
    int count = 0;
    for (int s = mine.x; s < mine.y; ++s) count += Child(a, s).copies(a, s);
    const int2 rank = team.scan<1>(count);                      // its barrier is behind the changes of the counts, unless there is one block
    if (team.ranks == 1) __syncthreads();
    const int got = list_free(a, team, rank.y);
    team.sync();
    int at = rank.x;
    for (int s = mine.x; s < mine.y; ++s) {
        const Child x(a, s);
        if (!x.copies(a, s)) continue;
        const int to = at < got ? __ldcg(a.list + at) : -1;
        a.table[(int64_t)s * W + x.full] = to;
        if (to >= 0) {
            a.source[at] = a.t.table[(int64_t)x.parent * W + x.full];
            a.target[at] = to;
            a.refs[to] = 1;
        }
        ++at;
    }
    if (team.thread == 0) {
        *a.moves = got;
        *a.result = rank.y - got;
    }
}

// ---------------------------------------------------------------- compacting
// With L pages in use, those from L on move to the places below L that are free, in order.
__global__ void __launch_bounds__(kThreads) compact_kernel(const __grid_constant__ PageArgs a) {
    const Team team;
    let_next_begin();
    const int2 mine = warp_pages(a, team);
    auto live = [&](int i) { return a.t.refs[i] > 0; };
    const int2 rank = team.scan<0>(count_pages(mine, live));
    const int L = rank.y;
    const int2 hole = team.scan<1>(count_pages(mine, [&](int i) { return i < L && !live(i); }));
    const int low = L - hole.y;                                 // pages in use below L
    number_pages(mine, rank.x, live, [&](int i, bool on, int at) {
        if (on && i >= L) a.source[at - low] = i;
        if (!on && i < L) a.target[i - at] = i;                 // holes before it: places less pages in use
    });
    if (team.thread == 0) {
        *a.moves = hole.y;
        *a.result = L;
    }
    team.sync();
    number_pages(mine, rank.x, live, [&](int i, bool on, int at) {
        a.list[i] = !on ? -1 : i < L ? i : __ldcg(a.target + at - low);                      // where it goes
        a.refs[i] = i >= L ? 0 : a.t.refs[on ? i : __ldcg(a.source + i - at)];
    });
    team.sync();
    for_places(a, team, [](int) { return 0; }, [&](int, int, int, int64_t i, int e) { a.table[i] = is_page(a.t, e) ? __ldcg(a.list + e) : -1; });
}

// ---------------------------------------------------------------- copies
struct MoveArgs {
    ca_pool pools[kMovePools];
    int npools, chunks;                 // chunks of a page in the largest pool
    const int *source, *target, *moves;
};
constexpr int kMoveThreads = 256, kMoveUnroll = 8, kChunk = kMoveThreads * kMoveUnroll;     // pieces of 16 bytes

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveArgs a) {
    wait_for_previous();
    const int64_t units = (int64_t)*a.moves * a.npools * a.chunks;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int chunk = (int)(u % a.chunks), pool = (int)(u / a.chunks % a.npools);
        const int64_t m = u / a.chunks / a.npools;
        const ca_pool& p = a.pools[pool];
        const int row = p.row / 16, pieces = row * p.tokens * p.heads;
        const char* src = (const char*)p.data + a.source[m] * p.page;
        char* dst = (char*)p.data + a.target[m] * p.page;
        uint4 w[kMoveUnroll];
        int64_t at[kMoveUnroll];
#pragma unroll
        for (int k = 0; k < kMoveUnroll; ++k) {
            const int i = chunk * kChunk + k * kMoveThreads + threadIdx.x;
            const int r = i / row, h = r / p.tokens;
            at[k] = i < pieces ? (int64_t)(i - r * row) * 16 + (r - h * p.tokens) * p.token + h * p.head : -1;
            if (at[k] >= 0) w[k] = *reinterpret_cast<const uint4*>(src + at[k]);
        }
#pragma unroll
        for (int k = 0; k < kMoveUnroll; ++k)
            if (at[k] >= 0) *reinterpret_cast<uint4*>(dst + at[k]) = w[k];
    }
}

// ---------------------------------------------------------------- host
int check_table(const ca_table* t, bool lengths) {
    if (!t) { set_error("table is NULL"); return CA_ERR_NULL; }
    if (t->width < 0 || t->sequences < 0 || t->pages < 0) { set_error("width=%d sequences=%d pages=%d must not be negative", t->width, t->sequences, t->pages); return CA_ERR_BAD_DESC; }
    if (t->page < 16 || t->page % 16) { set_error("page=%d: multiples of 16 tokens are supported", t->page); return CA_ERR_BAD_DESC; }
    // 32-bit loops over them step by all threads of a cluster, and shares are rounded up
    if (t->pages > 1 << 30 || t->sequences > 1 << 30) { set_error("sequences=%d pages=%d exceed 2^30", t->sequences, t->pages); return CA_ERR_TOO_LARGE; }
    if ((int64_t)t->width * t->page > INT32_MAX) { set_error("width=%d places of %d tokens exceed 2^31 tokens", t->width, t->page); return CA_ERR_TOO_LARGE; }
    if ((t->sequences && t->width && !t->table) || (t->pages && !t->refs) || (lengths && t->sequences && !t->lengths)) { set_error("table, refs and lengths must not be NULL"); return CA_ERR_NULL; }
    return CA_OK;
}

int check_outputs(const ca_table* t, const int32_t* table, const int32_t* refs, const int32_t* result, const void* workspace) {
    if ((t->sequences && t->width && !table) || (t->pages && !refs) || !result || !workspace) { set_error("results and workspace must not be NULL"); return CA_ERR_NULL; }
    if (table && table == t->table) { set_error("the new table takes the old one's place"); return CA_ERR_BAD_DESC; }
    if (refs && refs == t->refs) { set_error("the new counts take the old ones' place"); return CA_ERR_BAD_DESC; }
    if (reinterpret_cast<uintptr_t>(workspace) % 16) { set_error("workspace is not 16-byte aligned"); return CA_ERR_BAD_DESC; }
    return CA_OK;
}

int check_pools(const ca_table* t, const ca_pool* pools, int npools) {
    if (npools < 0 || (npools && !pools)) { set_error("npools=%d without pools", npools); return CA_ERR_NULL; }
    for (int i = 0; i < npools; ++i) {
        const ca_pool& p = pools[i];
        if (t->pages && !p.data) { set_error("pool %d has no data (NULL)", i); return CA_ERR_NULL; }
        if (p.tokens != t->page) { set_error("pool %d has pages of %d tokens, the table of %d", i, p.tokens, t->page); return CA_ERR_BAD_DESC; }
        if (p.row < 16 || p.row % 16 || p.heads < 1) { set_error("pool %d: rows of %d bytes (multiples of 16 are supported), %d heads", i, p.row, p.heads); return CA_ERR_BAD_DESC; }
        if (reinterpret_cast<uintptr_t>(p.data) % 16 || p.token % 16 || p.head % 16 || p.page % 16 || p.token < 0 || p.head < 0 || p.page < 0) {
            set_error("pool %d: address and strides must be multiples of 16 bytes, strides not negative", i);
            return CA_ERR_BAD_DESC;
        }
        if ((int64_t)p.row / 16 * p.tokens * p.heads > (1LL << 30)) { set_error("pool %d: pages of more than 16 GB", i); return CA_ERR_TOO_LARGE; }
    }
    return CA_OK;
}

// Lists of pages, then lists of sequences, then single numbers.
void split_workspace(PageArgs* a, void* workspace) {
    int* w = static_cast<int*>(workspace);
    a->moves = w;
    a->list = w + 4;
    a->source = a->list + a->t.pages;
    a->target = a->source + a->t.pages;
    a->keeper = a->target + a->t.pages;
    a->need = a->keeper;
    a->offset = a->keeper + a->t.sequences;
}

// Blocks of a cluster: 16 where the device schedules that, else the portable 8.  Cached per kernel and device.
template <typename K>
int most_blocks(K kernel, std::atomic<int>* cache) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (n) return n;
    n = 8;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = kBlocks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(kBlocks); cfg.blockDim = dim3(kThreads); cfg.attrs = at; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0) n = kBlocks;
    }
    cudaGetLastError();
    cache[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <void (*KERNEL)(const PageArgs)>
int launch_team(const PageArgs& a, cudaStream_t st, const char* name) {
    static std::atomic<int> cache[64];
    // Blocks that leave a thread four places or pages: a barrier of a larger cluster costs more (fork of 4352 places with 16 blocks
    // 15.3 us, with 8 12.9), fewer threads take longer (step over 85000 pages with 8 blocks 24.8 us, with 16 19.9).
    const int64_t things = std::max<int64_t>((int64_t)a.t.width * a.t.sequences, a.t.pages);
    int blocks = 1;
    while (blocks < kBlocks && things > 4LL * kThreads * blocks) blocks *= 2;
    blocks = std::min(blocks, blocks > 8 ? most_blocks(KERNEL, cache) : 8);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = blocks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(kThreads); cfg.stream = st;
    cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, a);
    if (e != cudaSuccess) return cuda_fail(e, name);
    CA_CHECK_LAUNCH(name);
    return CA_OK;
}

int launch_moves(const PageArgs& a, const ca_pool* pools, int npools, int64_t most, cudaStream_t st) {
    for (int first = 0; first < npools && most > 0; first += kMovePools) {
        MoveArgs m{};
        m.npools = std::min(kMovePools, npools - first);
        for (int i = 0; i < m.npools; ++i) {
            m.pools[i] = pools[first + i];
            m.chunks = std::max(m.chunks, (int)(((int64_t)m.pools[i].row / 16 * m.pools[i].tokens * m.pools[i].heads + kChunk - 1) / kChunk));
        }
        m.source = a.source;
        m.target = a.target;
        m.moves = a.moves;
        const int64_t units = most * m.npools * m.chunks;
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = first == 0;
        cfg.gridDim = dim3((unsigned)std::min<int64_t>(units, 8LL * sm_count())); cfg.blockDim = dim3(kMoveThreads); cfg.stream = st;
        cfg.attrs = at; cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, move_kernel, m);
        if (e != cudaSuccess) return cuda_fail(e, "page copy kernel");
        CA_CHECK_LAUNCH("page copy kernel");
    }
    return CA_OK;
}

}  // namespace
}  // namespace ca

using namespace ca;

extern "C" {

size_t ca_pages_workspace(const ca_table* t) {
    if (check_table(t, false)) return 0;
    return ((size_t)4 + 3 * (size_t)t->pages + (1 + kBlocks) * (size_t)t->sequences) * sizeof(int32_t);
}

int ca_advance_pages(const ca_table* t, const int32_t* starts, int32_t left, int32_t sinks, int32_t* table, int32_t* refs, int32_t* missing,
                     void* workspace, void* stream) {
    int rc = check_table(t, true);
    if (rc || (rc = check_outputs(t, table, refs, missing, workspace))) return rc;
    if (sinks < 0) { set_error("sinks=%d must not be negative", sinks); return CA_ERR_BAD_DESC; }
    if (t->sequences && !starts) { set_error("starts must not be NULL"); return CA_ERR_NULL; }
    PageArgs a{};
    a.t = *t;
    a.starts = starts;
    a.left = left;
    a.sinks = sinks;
    a.table = table; a.refs = refs; a.result = missing;
    split_workspace(&a, workspace);
    return launch_team<advance_kernel>(a, as_stream(stream), "page step kernel");
}

int ca_fork_pages(const ca_table* t, const int32_t* parents, const ca_pool* pools, int32_t npools, int32_t* table, int32_t* refs,
                  int32_t* lengths, int32_t* missing, void* workspace, void* stream) {
    int rc = check_table(t, true);
    if (rc || (rc = check_outputs(t, table, refs, missing, workspace)) || (rc = check_pools(t, pools, npools))) return rc;
    if (t->sequences && (!parents || !lengths)) { set_error("parents and lengths must not be NULL"); return CA_ERR_NULL; }
    if (lengths && lengths == t->lengths) { set_error("the new lengths take the old ones' place"); return CA_ERR_BAD_DESC; }
    PageArgs a{};
    a.t = *t;
    a.parents = parents;
    a.table = table; a.refs = refs; a.lengths = lengths; a.result = missing;
    split_workspace(&a, workspace);
    rc = launch_team<fork_kernel>(a, as_stream(stream), "page fork kernel");
    return rc ? rc : launch_moves(a, pools, npools, std::min(t->sequences, t->pages), as_stream(stream));
}

int ca_compact_pages(const ca_table* t, const ca_pool* pools, int32_t npools, int32_t* table, int32_t* refs, int32_t* live,
                     void* workspace, void* stream) {
    int rc = check_table(t, false);
    if (rc || (rc = check_outputs(t, table, refs, live, workspace)) || (rc = check_pools(t, pools, npools))) return rc;
    PageArgs a{};
    a.t = *t;
    a.table = table; a.refs = refs; a.result = live;
    split_workspace(&a, workspace);
    rc = launch_team<compact_kernel>(a, as_stream(stream), "page compaction kernel");
    return rc ? rc : launch_moves(a, pools, npools, t->pages / 2, as_stream(stream));
}

}  // extern "C"
