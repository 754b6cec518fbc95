// Attention over a paged cache for few query rows a key head: decoding, and short chunks.
//
// Bound: the bytes of the visible keys and values, read once.  A tile of 128 query rows would be mostly empty here, and what
// counts is how many bytes are under way; so each warp runs for itself.  It takes tiles of 16 keys (pages are multiples of 16
// tokens, so a tile lies in one page), copies the next ones with cp.async while it works on one, and keeps its own running
// maximum, sum and accumulator for 16 rows; no thread waits for another warp before the end.  16-bit types multiply on
// m16n8k16 (tcgen05 works on 128 rows), Float32 on the FMA pipe.
//
// The keys of a sequence and key head are split over a cluster of up to 16 CTAs, whose parts are joined through distributed
// shared memory in a fixed order: one launch, no scratch memory.
//
// Measured: 64 sequences, windows of 4096 tokens, 32 query and 8 key heads of 128 features, bfloat16 (1.08 GB): 182 us, 5.9 TB/s,
// 0.91 of a copy's rate; Float32 (2.16 GB) 719 us, 3.0 TB/s.  4 sequences of up to 3000 tokens (17 MB): 13.7 us on 128 CTAs, in
// clusters of 8: the bound on row tiles (paged_tiles) counts 5 for 4, and the split ends where it takes those for more than fill
// the chip.
#include <cooperative_groups.h>
#include <algorithm>

#include "seq_umma.cuh"

namespace cg = cooperative_groups;

namespace ca {
namespace {

constexpr int kWarps = 4, kKeys = 16, kRows = 16;

template <typename T, int DM> struct Decode {
    static constexpr int kRowBytes = DM * sizeof(T), kPieces = kRowBytes / 16;
    static constexpr int kStages = 3;
    static constexpr int kStageBytes = 2 * kKeys * kRowBytes;                       // keys, then values
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kParts = kWarps * kRows * DM * 4;                          // in the ring's place at the end
    static constexpr int kQuery = sizeof(T) == 4 ? kRows * DM * 4 + kWarps * kRows * kKeys * 4 : 0;   // queries and weights in Float32
    static constexpr size_t kSmem = (kRing > kParts ? kRing : kParts) + kQuery;
    // piece c of row r: eight rows of one piece, or eight pieces of one row, lie in different banks
    static __device__ __forceinline__ int at(int r, int c) { return r * kRowBytes + ((c & ~7 | ((c ^ r) & 7)) << 4); }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load4_turned(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (kIsBf16<T>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Row maxima that a warp has in registers grow by at least 2^8 before its accumulator is rescaled.
__device__ __forceinline__ bool grows(float& m, float top, float& f) {
    f = 1.f;
    if (!(top > m + 8.f)) return false;
    f = fast_exp2(m - top);
    m = top;
    return true;
}

template <typename T, int DM>
__global__ void __launch_bounds__(32 * kWarps) decode_kernel(const __grid_constant__ SeqArgs a) {
    typedef Decode<T, DM> L;
    extern __shared__ __align__(128) char smem[];
    __shared__ float part_m[kWarps][kRows], part_l[kWarps][kRows], row_m[kRows], row_l[kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.y;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    int tile = (int)blockIdx.x / ranks;
    const int2 owned = owned_tokens(a);
    Seq s;
    if (!paged_seq(a, kRows, tile, &s)) {                          // alike in the whole cluster
        clear_unowned<T>(a, owned, h, tid, 32 * kWarps);
        return;
    }
    const int rows = s.T * a.G, R0 = tile * kRows, nrows = min(kRows, rows - R0);
    const int p_lo = s.base + R0 / a.G, p_hi = s.base + (R0 + nrows - 1) / a.G;
    const KeyTiles kt = key_tiles(a, s, p_lo, p_hi, kKeys);
    const int first = (int)((int64_t)kt.count * rank / ranks), last = (int)((int64_t)kt.count * (rank + 1) / ranks);
    const int c_lo = max(p_lo, 0) - a.left, c_hi = min(p_hi, s.n - 1);        // keys that any row sees (or < sinks)

    // ------------------------------------------------------------ copies: tile i of this warp into stage `st`
    const uint32_t ring = smem_u32(smem) + warp * L::kStages * L::kStageBytes;
    const int piece = lane % L::kPieces, row0 = lane / L::kPieces, feature = piece * (16 / (int)sizeof(T));
    constexpr int STEP = 32 / L::kPieces > 0 ? 32 / L::kPieces : 1;
    const char* const k_lane = (const char*)((const T*)a.kp.data + h * a.kp.head + row0 * a.kp.token + feature);
    const char* const v_lane = (const char*)((const T*)a.vp.data + h * a.vp.head + row0 * a.vp.token + feature);
    const int64_t k_step = STEP * a.kp.token * (int64_t)sizeof(T), v_step = STEP * a.vp.token * (int64_t)sizeof(T);
    auto copy_tile = [&](int i, int st, int page) {
        if (page >= 0) {
            const int key0 = kt.key(i, kKeys), off = key0 % a.pages.page;
            const char* k = k_lane + (off * a.kp.token + page * a.kp.page) * (int64_t)sizeof(T);
            const char* v = v_lane + (off * a.vp.token + page * a.vp.page) * (int64_t)sizeof(T);
            const uint32_t to = ring + st * L::kStageBytes;
            const bool all = feature < a.D && key0 + kKeys - 1 <= c_hi && (key0 >= c_lo || key0 + kKeys <= a.sinks);
#pragma unroll
            for (int r = 0; r < kKeys; r += STEP, k += k_step, v += v_step) {
                const int j = key0 + r + row0;
                const bool on = all || (feature < a.D && j <= c_hi && (j >= c_lo || j < a.sinks));      // what no row sees counts as zeros
                copy16(to + L::at(r + row0, piece), on ? k : (const char*)a.kp.data, on);
                copy16(to + kKeys * L::kRowBytes + L::at(r + row0, piece), on ? v : (const char*)a.vp.data, on);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Pages of the warp's tiles, 32 at a time: lane k has that of tile first + warp + 4 (32 c + k), and those of the next 32
    // are on their way.
    auto page_at = [&](int n) {
        const int i = first + warp + kWarps * n;
        return i < last ? page_of(a, s.b, kt.key(i, kKeys)) : -1;
    };
    int page_now = page_at(lane), page_next = page_at(32 + lane);
    auto page = [&](int n) { return __shfl_sync(~0u, n & 32 ? page_next : page_now, n & 31); };      // n is at most 31 behind the first of now
#pragma unroll
    for (int st = 0; st < L::kStages - 1; ++st) copy_tile(first + warp + kWarps * st, st, page(st));
    clear_unowned<T>(a, owned, h, tid, 32 * kWarps);

    float m[sizeof(T) == 4 ? 8 : 2], l[sizeof(T) == 4 ? 8 : 2];
    constexpr int STATS = sizeof(T) == 4 ? 8 : 2;
#pragma unroll
    for (int i = 0; i < STATS; ++i) m[i] = -INFINITY, l[i] = 0.f;
    // body(tile in shared memory, key0) for each of the warp's tiles that exists
    auto for_tiles = [&](auto body) {
        int st = 0, ahead = L::kStages - 1, n = 0, first32 = 0;
        for (int i = first + warp; i < last; i += kWarps) {
            const int next = n + L::kStages - 1;
            copy_tile(first + warp + kWarps * (first32 + next), ahead, page(next));
            const int now = page(n);
            asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
            __syncwarp();
            if (now >= 0) body(smem + warp * L::kStages * L::kStageBytes + st * L::kStageBytes, kt.key(i, kKeys));
            __syncwarp();
            st = st + 1 == L::kStages ? 0 : st + 1;
            ahead = ahead + 1 == L::kStages ? 0 : ahead + 1;
            if (++n == 32) {                                    // numbers count from the first of these 32 tiles
                n = 0;
                first32 += 32;
                page_now = page_next;
                page_next = page_at(first32 + 32 + lane);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    };
    float* const parts = reinterpret_cast<float*>(smem) + warp * kRows * DM;       // [warp][row][feature] at the end

    if constexpr (sizeof(T) == 2) {
        const int ra = lane >> 2, pa = s.base + token_of(a, min(R0 + ra, rows - 1)), pb = s.base + token_of(a, min(R0 + ra + 8, rows - 1));
        uint32_t q[DM / 16][4];
        {
            const T* qa = ra < nrows ? seq_row<T>(a.q, a, s, h, R0 + ra) : nullptr;
            const T* qb = ra + 8 < nrows ? seq_row<T>(a.q, a, s, h, R0 + ra + 8) : nullptr;
#pragma unroll
            for (int k = 0; k < DM / 16; ++k) {
                const int f = k * 16 + (lane & 3) * 2;
                q[k][0] = qa && f < a.D ? *reinterpret_cast<const uint32_t*>(qa + f) : 0u;
                q[k][1] = qb && f < a.D ? *reinterpret_cast<const uint32_t*>(qb + f) : 0u;
                q[k][2] = qa && f + 8 < a.D ? *reinterpret_cast<const uint32_t*>(qa + f + 8) : 0u;
                q[k][3] = qb && f + 8 < a.D ? *reinterpret_cast<const uint32_t*>(qb + f + 8) : 0u;
            }
        }
        float o[DM / 8][4];
#pragma unroll
        for (int i = 0; i < DM / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for_tiles([&](char* tile_at, int key0) {
            const uint32_t ks = smem_u32(tile_at), vs = ks + kKeys * L::kRowBytes;
            float c[2][4] = {};
#pragma unroll
            for (int k = 0; k < DM / 16; ++k) {
                uint32_t b[4];                                  // keys 0-7 and 8-15, features 16k .. 16k+7 and +8 .. +15
                load4(b, ks + L::at((lane >> 4) * 8 + (lane & 7), 2 * k + (lane >> 3 & 1)));
                mma16<T>(c[0], q[k], b[0], b[1]);
                mma16<T>(c[1], q[k], b[2], b[3]);
            }
            const int j = key0 + (lane & 3) * 2;
            const bool edge = !(p_lo >= 0 && key0 + kKeys - 1 <= p_lo && (key0 >= p_hi - a.left || key0 + kKeys <= a.sinks));
            float ta = -INFINITY, tb = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[n][e] *= a.scale_log2;
                    if (edge && !sees(a, s.n, e < 2 ? pa : pb, j + 8 * n + (e & 1))) c[n][e] = -INFINITY;
                    if (e < 2) ta = fmaxf(ta, c[n][e]); else tb = fmaxf(tb, c[n][e]);
                }
            ta = fmaxf(ta, __shfl_xor_sync(~0u, ta, 1));
            tb = fmaxf(tb, __shfl_xor_sync(~0u, tb, 1));
            ta = fmaxf(ta, __shfl_xor_sync(~0u, ta, 2));
            tb = fmaxf(tb, __shfl_xor_sync(~0u, tb, 2));
            float fa, fb;
            const bool grew = grows(m[0], ta, fa) | grows(m[1], tb, fb);
            if (__any_sync(~0u, grew)) {
                l[0] *= fa;
                l[1] *= fb;
#pragma unroll
                for (int i = 0; i < DM / 8; ++i) { o[i][0] *= fa; o[i][1] *= fa; o[i][2] *= fb; o[i][3] *= fb; }
            }
            const float ma = m[0] == -INFINITY ? 0.f : m[0], mb = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[n][e] = fast_exp2(c[n][e] - (e < 2 ? ma : mb));
            l[0] += (c[0][0] + c[0][1]) + (c[1][0] + c[1][1]);
            l[1] += (c[0][2] + c[0][3]) + (c[1][2] + c[1][3]);
            const uint32_t p[4] = {pack16<T>(c[0][0], c[0][1]), pack16<T>(c[0][2], c[0][3]), pack16<T>(c[1][0], c[1][1]), pack16<T>(c[1][2], c[1][3])};
#pragma unroll
            for (int i = 0; i < DM / 16; ++i) {
                uint32_t b[4];                                  // keys 0-7 and 8-15 of features 16i .. +7, then of the next 8
                load4_turned(b, vs + L::at((lane >> 3 & 1) * 8 + (lane & 7), 2 * i + (lane >> 4)));
                mma16<T>(o[2 * i], p, b[0], b[1]);
                mma16<T>(o[2 * i + 1], p, b[2], b[3]);
            }
        });
        __syncthreads();                                        // the ring is free
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(~0u, l[i], 1);
            l[i] += __shfl_xor_sync(~0u, l[i], 2);
            if ((lane & 3) == 0) {
                part_m[warp][ra + 8 * i] = m[i];
                part_l[warp][ra + 8 * i] = l[i];
            }
        }
#pragma unroll
        for (int i = 0; i < DM / 8; ++i) {
            *reinterpret_cast<float2*>(parts + ra * DM + 8 * i + (lane & 3) * 2) = make_float2(o[i][0], o[i][1]);
            *reinterpret_cast<float2*>(parts + (ra + 8) * DM + 8 * i + (lane & 3) * 2) = make_float2(o[i][2], o[i][3]);
        }
    } else {
        // Float32: lane = key and every second row for the scores, lane = DM/32 features for the weighted sum
        constexpr int C = DM / 32;
        float* const Q = reinterpret_cast<float*>(smem + (L::kRing > L::kParts ? L::kRing : L::kParts));
        float* const P = Q + kRows * DM + warp * kRows * kKeys;
        for (int i = tid; i < kRows * DM; i += 32 * kWarps) {
            const int r = i / DM, f = i % DM;
            Q[i] = r < nrows && f < a.D ? seq_row<float>(a.q, a, s, h, R0 + min(r, nrows - 1))[f] : 0.f;
        }
        __syncthreads();
        const int half = lane >> 4, key = lane & 15;
        int pos[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pos[i] = 2 * i + half < nrows ? s.base + token_of(a, R0 + 2 * i + half) : -1;
        float o[kRows][C];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) o[r][c] = 0.f;
        for_tiles([&](char* tile_at, int key0) {
            const char *ks = tile_at, *vs = tile_at + kKeys * L::kRowBytes;
            float sc[8];
#pragma unroll
            for (int g = 0; g < 8; g += 2) {
                sc[g] = sc[g + 1] = 0.f;
                if (2 * g >= nrows) continue;
                f32x2 x = 0, y = 0;
#pragma unroll 4
                for (int c = 0; c < DM / 4; ++c) {
                    const ulonglong2 kk = *reinterpret_cast<const ulonglong2*>(ks + L::at(key, c));
                    const ulonglong2 qx = *reinterpret_cast<const ulonglong2*>(Q + (2 * g + half) * DM + 4 * c);
                    const ulonglong2 qy = *reinterpret_cast<const ulonglong2*>(Q + (2 * g + 2 + half) * DM + 4 * c);
                    x = fma2(qx.y, kk.y, fma2(qx.x, kk.x, x));
                    y = fma2(qy.y, kk.y, fma2(qy.x, kk.x, y));
                }
                float x0, x1, y0, y1;
                unpack2(x, x0, x1);
                unpack2(y, y0, y1);
                sc[g] = x0 + x1;
                sc[g + 1] = y0 + y1;
            }
            float f[8];
            bool grew = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = 1.f;
                if (2 * i >= nrows) continue;
                sc[i] = sees(a, s.n, pos[i], key0 + key) ? sc[i] * a.scale_log2 : -INFINITY;
                float top = sc[i];
#pragma unroll
                for (int x = 8; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
                grew |= grows(m[i], top, f[i]);
                l[i] *= f[i];
                const float p = fast_exp2(sc[i] - (m[i] == -INFINITY ? 0.f : m[i]));
                l[i] += p;
                P[(2 * i + half) * kKeys + key] = p;
            }
            if (__any_sync(~0u, grew)) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if (r >= nrows) break;
                    const float g = __shfl_sync(~0u, f[r >> 1], (r & 1) * 16);
#pragma unroll
                    for (int c = 0; c < C; ++c) o[r][c] *= g;
                }
            }
            __syncwarp();
#pragma unroll 1
            for (int k = 0; k < kKeys; k += 4) {
                float v[4][C];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float* src = reinterpret_cast<const float*>(vs + L::at(k + e, lane * C / 4)) + lane * C % 4;
#pragma unroll
                    for (int c = 0; c < C; ++c) v[e][c] = src[c];
                }
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if (r >= nrows) break;
                    const float4 p = *reinterpret_cast<const float4*>(P + r * kKeys + k);
#pragma unroll
                    for (int c = 0; c < C; ++c) o[r][c] = fmaf(p.x, v[0][c], fmaf(p.y, v[1][c], fmaf(p.z, v[2][c], fmaf(p.w, v[3][c], o[r][c]))));
                }
            }
        });
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float sum = l[i];
#pragma unroll
            for (int x = 8; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
            if (key == 0) {
                part_m[warp][2 * i + half] = m[i];
                part_l[warp][2 * i + half] = sum;
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c) parts[r * DM + lane * C + c] = o[r][c];
    }

    // ------------------------------------------------------------ join: the CTA's warps, then the CTAs; four features a thread
    __syncthreads();
    auto put = [&](int r, int f, float4 y, float sum) {
        if (f >= a.D) return;
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        if (sum == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);    // sees nothing: zeros, next to infinities too
        T* dst = seq_row<T>(a.y, a, s, h, R0 + r) + f;
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<T>(y.x * inv, y.y * inv), pack16<T>(y.z * inv, y.w * inv));
        else
            *reinterpret_cast<float4*>(dst) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    };
    auto add = [](float4& y, float4 x, float g) { y.x = fmaf(x.x, g, y.x); y.y = fmaf(x.y, g, y.y); y.z = fmaf(x.z, g, y.z); y.w = fmaf(x.w, g, y.w); };
    const int items = nrows * (DM / 4);
    float* const all = reinterpret_cast<float*>(smem);          // [warp][row][feature]; the sum takes the first warp's place
    for (int i = tid; i < items; i += 32 * kWarps) {
        const int r = i / (DM / 4), f = i % (DM / 4) * 4;
        float M = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, part_m[w][r]);
        const float ref = M == -INFINITY ? 0.f : M;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float g = fast_exp2(part_m[w][r] - ref);
            sum = fmaf(part_l[w][r], g, sum);
            add(y, *reinterpret_cast<const float4*>(all + (w * kRows + r) * DM + f), g);
        }
        if (ranks == 1) {
            put(r, f, y, sum);
        } else {
            *reinterpret_cast<float4*>(all + r * DM + f) = y;
            if (f == 0) { row_m[r] = M; row_l[r] = sum; }
        }
    }
    if (ranks == 1) return;
    cluster.sync();
    const int begin = items * rank / ranks, end = items * (rank + 1) / ranks;
    for (int i = begin + tid; i < end; i += 32 * kWarps) {
        const int r = i / (DM / 4), f = i % (DM / 4) * 4;
        float M = -INFINITY, sum = 0.f;
#pragma unroll 4
        for (int c = 0; c < ranks; ++c) M = fmaxf(M, *cluster.map_shared_rank(&row_m[r], c));
        const float ref = M == -INFINITY ? 0.f : M;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < ranks; ++c) {
            const float g = fast_exp2(*cluster.map_shared_rank(&row_m[r], c) - ref);
            sum = fmaf(*cluster.map_shared_rank(&row_l[r], c), g, sum);
            add(y, *reinterpret_cast<const float4*>(cluster.map_shared_rank(all + r * DM + f, c)), g);
        }
        put(r, f, y, sum);
    }
    cluster.sync();                                             // nobody leaves while its part is read
}

// Largest cluster of the kernel that the device schedules (16 where it can, else the portable 8).  Cached per kernel and
// device: a function's attributes are those of the current device.
template <typename K>
int largest_cluster(K kernel, size_t smem, std::atomic<int>* cache) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (n) return n;
    n = 8;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 16; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(16); cfg.blockDim = dim3(32 * kWarps); cfg.dynamicSmemBytes = smem; cfg.attrs = at; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0) n = 16;
    }
    cudaGetLastError();
    cache[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <typename T, int DM>
int launch(const SeqArgs& a, cudaStream_t st) {
    static std::atomic<int> cluster_cache[64];
    const size_t smem = Decode<T, DM>::kSmem;
    cudaError_t e = cudaFuncSetAttribute(decode_kernel<T, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    const int64_t tiles = paged_tiles(a.N, a.G, a.pages.sequences, kRows);
    // Split the keys while that fills idle SMs (two CTAs each) and leaves every warp a few tiles.  What is known here is the
    // most keys that a row can see: the table's width, or the window with the first tokens.
    const int64_t keys = std::min<int64_t>((int64_t)a.pages.width * a.pages.page, (int64_t)a.left + a.sinks + a.N);
    const int most = largest_cluster(decode_kernel<T, DM>, smem, cluster_cache);
    int split = 1;
    while (split < most && tiles * a.Hkv * split * 2 <= 2LL * sm_count() && keys >= (int64_t)split * 2 * kWarps * kKeys * 2) split *= 2;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * split), a.Hkv, 1); cfg.blockDim = dim3(32 * kWarps); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = at; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, decode_kernel<T, DM>, a);
    if (e != cudaSuccess) return cuda_fail(e, "paged decode kernel");
    CA_CHECK_LAUNCH("paged decode kernel");
    return CA_OK;
}

}  // namespace

int decode_paged(const SeqArgs& a, int dtype, cudaStream_t st) {
    const bool wide = a.D > 64;
    if (dtype == CA_F32) return wide ? launch<float, 128>(a, st) : launch<float, 64>(a, st);
    if (dtype == CA_BF16) return wide ? launch<__nv_bfloat16, 128>(a, st) : launch<__nv_bfloat16, 64>(a, st);
    return wide ? launch<__half, 128>(a, st) : launch<__half, 64>(a, st);
}

}  // namespace ca
