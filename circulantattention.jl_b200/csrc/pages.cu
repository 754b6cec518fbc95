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
#include <cooperative_groups.h>
#include <algorithm>
#include "seq.cuh"

namespace cg = cooperative_groups;

namespace ca {
namespace {

constexpr int kThreads = 1024, kBlocks = 8, kMovePools = 32;

struct PageArgs {
    ca_table t;
    const int *starts, *parents;
    int left, sinks;
    int *table, *refs, *lengths, *result;       // the next state; result: pages that were wanting, or pages in use
    int *list, *source, *target, *keeper, *offset, *moves;
};

struct Team {
    cg::cluster_group cluster;
    int thread, threads, rank, ranks;
    __device__ __forceinline__ Team() : cluster(cg::this_cluster()), rank((int)cluster.block_rank()), ranks((int)cluster.num_blocks()) {
        thread = rank * kThreads + threadIdx.x;
        threads = ranks * kThreads;
    }
    // Everything that the cluster's threads wrote before is seen behind this
    __device__ __forceinline__ void sync() const {
        __threadfence();
        cluster.sync();
    }
    // Sum of v over the threads before this one, and over all of them
    __device__ int2 scan(int v) const {
        __shared__ int warps[kThreads / 32], block;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        int upto = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) warps[warp] = upto;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += warps[w];
            all += warps[w];
        }
        if (threadIdx.x == 0) block = all;
        cluster.sync();
        int total = 0;
        for (int r = 0; r < ranks; ++r) {
            const int x = *cluster.map_shared_rank(&block, r);
            if (r < rank) before += x;
            total += x;
        }
        cluster.sync();                                         // the totals have been read
        return make_int2(before + upto - v, total);
    }
};

// This thread's share of n consecutive things
__device__ __forceinline__ int2 share(const Team& team, int n) {
    const int piece = (n + team.threads - 1) / team.threads;
    const int64_t at = (int64_t)piece * team.thread;
    return make_int2((int)min((int64_t)n, at), (int)min((int64_t)n, at + piece));
}

__device__ __forceinline__ bool is_page(const ca_table& t, int e) { return e >= 0 && e < t.pages; }

// Lists the lowest `wanted` pages without users; returns how many of them there are.
__device__ int list_free(const PageArgs& a, const Team& team, int wanted) {
    const int2 mine = share(team, a.t.pages);
    int count = 0;
    for (int i = mine.x; i < mine.y; ++i) count += __ldcg(a.refs + i) <= 0;
    const int2 rank = team.scan(count);
    int at = rank.x;
    for (int i = mine.x; i < mine.y && at < wanted; ++i)
        if (__ldcg(a.refs + i) <= 0) a.list[at++] = i;
    return min(rank.y, wanted);
}

// ---------------------------------------------------------------- a serving step
// What stays of sequence s: the places first..upto - 1 and those below `sinks`; new tokens are in fresh..upto - 1.
struct Stay {
    int first, upto, sinks, fresh;
    __device__ __forceinline__ Stay(const PageArgs& a, int s) {
        const int page = a.t.page;
        const int64_t n = max(0, a.t.lengths[s]), count = (int64_t)a.starts[s + 1] - a.starts[s];
        const int64_t begin = max((int64_t)0, n - max((int64_t)0, count));
        upto = (int)min((int64_t)a.t.width, (n + page - 1) / page);
        first = a.left < 0 ? 0 : (int)(max((int64_t)0, begin - a.left) / page);
        sinks = (int)((min((int64_t)a.sinks, n) + page - 1) / page);
        fresh = count > 0 ? (int)min((int64_t)upto, begin / page) : upto;
    }
    __device__ __forceinline__ bool has(int c) const { return c < upto && (c >= first || c < sinks); }
};

__global__ void __launch_bounds__(kThreads) advance_kernel(const __grid_constant__ PageArgs a) {
    const Team team;
    const int S = a.t.sequences, W = a.t.width, lane = threadIdx.x & 31;
    for (int i = team.thread; i < a.t.pages; i += team.threads) a.refs[i] = a.t.refs[i];
    team.sync();
    for (int64_t i = team.thread; i < (int64_t)S * W; i += team.threads) {
        const int s = (int)(i / W), c = (int)(i - (int64_t)s * W), e = a.t.table[i];
        const bool there = is_page(a.t, e), stays = Stay(a, s).has(c);
        a.table[i] = there && stays ? e : -1;
        if (there && !stays) atomicSub(a.refs + e, 1);
    }
    // a warp for each sequence: its new places without a page
    int wanted = 0;
    for (int s = team.thread >> 5; s < S; s += team.threads >> 5) {
        const Stay stay(a, s);
        int need = 0;
        for (int c = stay.fresh + lane; c < stay.upto; c += 32) need += !is_page(a.t, a.t.table[(int64_t)s * W + c]);
        need = __reduce_add_sync(~0u, need);
        if (lane == 0) a.offset[s] = need;
        wanted += lane == 0 ? need : 0;
    }
    team.sync();
    // the sequences in order
    const int2 mine = share(team, S);
    int count = 0;
    for (int s = mine.x; s < mine.y; ++s) count += __ldcg(a.offset + s);
    int2 rank = team.scan(count);
    for (int s = mine.x; s < mine.y; ++s) {
        const int need = __ldcg(a.offset + s);
        a.offset[s] = rank.x;
        rank.x += need;
    }
    const int got = list_free(a, team, rank.y);
    team.sync();
    for (int s = team.thread >> 5; s < S; s += team.threads >> 5) {
        const Stay stay(a, s);
        int at = __ldcg(a.offset + s);
        for (int c0 = stay.fresh; c0 < stay.upto; c0 += 32) {
            const int c = c0 + lane;
            const bool need = c < stay.upto && !is_page(a.t, a.t.table[(int64_t)s * W + c]);
            const unsigned all = __ballot_sync(~0u, need);
            const int k = at + __popc(all & ((1u << lane) - 1));
            if (need && k < got) {
                const int p = __ldcg(a.list + k);
                a.table[(int64_t)s * W + c] = p;
                a.refs[p] = 1;
            }
            at += __popc(all);
        }
    }
    if (team.thread == 0) *a.result = rank.y - got;
}

// ---------------------------------------------------------------- forking
__device__ __forceinline__ int parent_of(const PageArgs& a, int s) {
    const int p = a.parents[s];
    return p >= 0 && p < a.t.sequences ? p : -1;
}
__device__ __forceinline__ int length_of(const PageArgs& a, int p) {
    return p < 0 ? 0 : (int)min((int64_t)max(0, a.t.lengths[p]), (int64_t)a.t.width * a.t.page);
}
// Whether sequence s needs a copy of its parent's last page: it is partly filled, and another sequence keeps it.
__device__ __forceinline__ bool wants_copy(const PageArgs& a, int s, int p, int n) {
    return p >= 0 && p != s && n % a.t.page && __ldcg(a.keeper + p) != s && is_page(a.t, a.t.table[(int64_t)p * a.t.width + n / a.t.page]);
}

__global__ void __launch_bounds__(kThreads) fork_kernel(const __grid_constant__ PageArgs a) {
    const Team team;
    const int S = a.t.sequences, W = a.t.width, page = a.t.page;
    for (int i = team.thread; i < a.t.pages; i += team.threads) a.refs[i] = a.t.refs[i];
    for (int s = team.thread; s < S; s += team.threads) a.keeper[s] = S;
    team.sync();
    // the partly filled page stays with the parent if it goes on, else with the first sequence that continues it
    for (int s = team.thread; s < S; s += team.threads) {
        const int p = parent_of(a, s);
        if (p >= 0) atomicMin(a.keeper + p, p == s ? -1 : s);
        a.lengths[s] = p < 0 ? 0 : a.t.lengths[p];
    }
    team.sync();
    for (int64_t i = team.thread; i < (int64_t)S * W; i += team.threads) {
        const int s = (int)(i / W), c = (int)(i - (int64_t)s * W), p = parent_of(a, s), old = a.t.table[i];
        int e = old;
        if (p != s) {
            if (is_page(a.t, old)) atomicSub(a.refs + old, 1);
            const int n = length_of(a, p), full = n / page;
            e = -1;
            if (c < full || (c == full && n % page && __ldcg(a.keeper + p) == s)) {
                e = a.t.table[(int64_t)p * W + c];
                if (is_page(a.t, e)) atomicAdd(a.refs + e, 1);
                else e = -1;
            }
        }
        a.table[i] = e;
    }
    const int2 mine = share(team, S);
    int count = 0;
    for (int s = mine.x; s < mine.y; ++s) {
        const int p = parent_of(a, s);
        count += wants_copy(a, s, p, length_of(a, p));
    }
    team.sync();
    const int2 rank = team.scan(count);
    const int got = list_free(a, team, rank.y);
    team.sync();
    int at = rank.x;
    for (int s = mine.x; s < mine.y; ++s) {
        const int p = parent_of(a, s), n = length_of(a, p);
        if (!wants_copy(a, s, p, n)) continue;
        if (at < got) {
            const int to = __ldcg(a.list + at);
            a.source[at] = a.t.table[(int64_t)p * W + n / page];
            a.target[at] = to;
            a.table[(int64_t)s * W + n / page] = to;
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
    const int S = a.t.sequences, W = a.t.width;
    const int2 mine = share(team, a.t.pages);
    int count = 0;
    for (int i = mine.x; i < mine.y; ++i) count += a.t.refs[i] > 0;
    const int2 rank = team.scan(count);
    const int L = rank.y;
    int holes = 0;
    for (int i = mine.x; i < mine.y; ++i) holes += i < L && a.t.refs[i] <= 0;
    const int2 hole = team.scan(holes);
    // pages in use below L: L less the holes
    int used = rank.x, free = hole.x;
    for (int i = mine.x; i < mine.y; ++i) {
        const bool live = a.t.refs[i] > 0;
        if (live && i >= L) a.source[used - (L - hole.y)] = i;
        if (!live && i < L) a.target[free++] = i;
        used += live;
    }
    team.sync();
    used = rank.x;
    free = hole.x;
    for (int i = mine.x; i < mine.y; ++i) {
        const int r = a.t.refs[i];
        const bool live = r > 0;
        a.list[i] = !live ? -1 : i < L ? i : __ldcg(a.target + used - (L - hole.y));     // where it goes
        a.refs[i] = i >= L ? 0 : live ? r : a.t.refs[__ldcg(a.source + free++)];
        used += live;
    }
    team.sync();
    for (int64_t i = team.thread; i < (int64_t)S * W; i += team.threads) {
        const int e = a.t.table[i];
        a.table[i] = is_page(a.t, e) ? __ldcg(a.list + e) : -1;
    }
    if (team.thread == 0) {
        *a.moves = hole.y;
        *a.result = L;
    }
}

// ---------------------------------------------------------------- copies
struct MoveArgs {
    ca_pool pools[kMovePools];
    int npools, chunks;                 // chunks of a page in the largest pool
    const int *source, *target, *moves;
};
constexpr int kMoveThreads = 256, kMoveUnroll = 8, kChunk = kMoveThreads * kMoveUnroll;     // pieces of 16 bytes

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const __grid_constant__ MoveArgs a) {
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
    a->offset = a->keeper + a->t.sequences;
}

template <typename K>
int launch_team(K kernel, const PageArgs& a, cudaStream_t st, const char* name) {
    // One block where that has a thread for every place and page
    const int64_t things = std::max<int64_t>((int64_t)a.t.width * a.t.sequences, a.t.pages);
    const int blocks = things <= 2 * kThreads ? 1 : kBlocks;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = blocks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(kThreads); cfg.stream = st;
    cfg.attrs = at; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
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
        move_kernel<<<(unsigned)std::min<int64_t>(units, 8LL * sm_count()), kMoveThreads, 0, st>>>(m);
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
    return ((size_t)4 + 3 * (size_t)t->pages + 2 * (size_t)t->sequences) * sizeof(int32_t);
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
    return launch_team(advance_kernel, a, as_stream(stream), "page step kernel");
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
    rc = launch_team(fork_kernel, a, as_stream(stream), "page fork kernel");
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
    rc = launch_team(compact_kernel, a, as_stream(stream), "page compaction kernel");
    return rc ? rc : launch_moves(a, pools, npools, t->pages / 2, as_stream(stream));
}

}  // extern "C"
