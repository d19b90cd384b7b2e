// Scaled Gaussian embedding lookup, and its gradient over tokens sorted by id.
//
//   forward   mz[t] = s mw[id_t],  Sz[t] = s^2 Sw[id_t]
//   gradient  g_m[v] = s sum_{t: id_t = v} dm[t],  g_S[v] = s^2 sum dS[t]
//
// The scan of embedding.cu reads every id once per vocabulary row, V x n compares:
// right for tens of rows, hopeless for the tens of thousands of a text vocabulary.
// Here the tokens are first sorted by id (a stable radix sort of (id, position)
// by one cluster), so that a row's tokens are neighbours and its sum is a
// segment of the sorted list:
//
//   sort    1 launch.  One cluster; each pass takes up to 8 bits of the id.
//   reduce  1 launch.  Block (c, slice) walks the kChunk tokens of chunk c over
//           its columns. A segment inside the chunk is finished at once; one that
//           crosses a border leaves a partial sum (head: it began earlier; tail:
//           it began here and goes on), and the chunk of a tail is put on a list.
//           Further blocks zero the rows that no token names (sums, deltas).
//   join    1 launch.  A block takes listed chunks and adds the heads that follow.
//
// Chunks are cut by position alone and partials are added in chunk order, so the
// result does not depend on scheduling. A row's tokens are added in token order
// within a chunk in fp32 and the chunks in double: a row that takes thousands of
// tokens loses no digits.
//
// Ids outside [0, V) and the padding id sort behind every row and are dropped.

#include <cooperative_groups.h>

#include <cstdint>

#include "common.cuh"
#include "tagi_b200.h"

namespace cg = cooperative_groups;

namespace tagi {
namespace {

enum { ID_F32 = 0, ID_I32 = 1, ID_I64 = 2 };

// The row of a token id, or -1. Float ids are truncated toward zero.
template <int IDT>
__device__ __forceinline__ int row_of(const void* ids, int64_t t, int V, int64_t pad) {
    if (IDT == ID_F32) {
        const float x = static_cast<const float*>(ids)[t];
        if (!(x > -1.0f && x < static_cast<float>(V))) return -1;
        const int v = static_cast<int>(x);
        return v == pad || v >= V ? -1 : v;
    }
    const int64_t v = IDT == ID_I32 ? static_cast<const int32_t*>(ids)[t]
                                    : static_cast<const int64_t*>(ids)[t];
    return v < 0 || v >= V || v == pad ? -1 : static_cast<int>(v);
}

template <int VEC>
struct Vec;
template <>
struct Vec<4> { using type = float4; };
template <>
struct Vec<2> { using type = float2; };
template <>
struct Vec<1> { using type = float; };

template <int VEC>
__device__ __forceinline__ void ldv(const float* p, float (&v)[VEC]) {
    // a plain load: the read-only path may not see what the kernel before this one, still
    // running when this one is launched, writes
    const typename Vec<VEC>::type x = *reinterpret_cast<const typename Vec<VEC>::type*>(p);
    const float* f = reinterpret_cast<const float*>(&x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = f[e];
}
// The same for values that are read once (the first to leave the caches: 84 us instead of
// 88 for the update below).
template <int VEC>
__device__ __forceinline__ void ldv_once(const float* p, float (&v)[VEC]) {
    const typename Vec<VEC>::type x = __ldcs(reinterpret_cast<const typename Vec<VEC>::type*>(p));
    const float* f = reinterpret_cast<const float*>(&x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = f[e];
}
template <int VEC>
__device__ __forceinline__ void stv(float* p, const float (&v)[VEC]) {
    typename Vec<VEC>::type x;
    float* f = reinterpret_cast<float*>(&x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = v[e];
    *reinterpret_cast<typename Vec<VEC>::type*>(p) = x;
}

// Bound by HBM: the named rows once, the outputs once. 16 bytes per thread and tensor
// where rows allow it. 16384 tokens x 512 of 32000 rows: 16.3 us, 5.2 TB/s of the bytes
// that have to move; a few tokens: the launch.
template <int VEC, int IDT>
__global__ void lookup_kernel(const void* ids, const float* mw, const float* Sw, float* mz,
                              float* Sz, int64_t n, int V, int D, int64_t pad, float s, float s2) {
    launch_dependents();
    const int per = D / VEC;
    const int64_t total = n * per;
    wait_for_primary();
    for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t t = i / per;
        const int j = static_cast<int>(i - t * per) * VEC;
        const int v = row_of<IDT>(ids, t, V, pad);
        float m[VEC], S[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.f;
        if (v >= 0) {
            ldv<VEC>(mw + static_cast<int64_t>(v) * D + j, m);
            ldv<VEC>(Sw + static_cast<int64_t>(v) * D + j, S);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                m[e] *= s;
                S[e] *= s2;
            }
        }
        stv<VEC>(mz + t * D + j, m);
        stv<VEC>(Sz + t * D + j, S);
    }
}

// ---- sort ---------------------------------------------------------------------
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kBins = 256;
constexpr int kSortCluster = 16;  // above the portable 8: scattered stores bind this kernel
constexpr int kItems = 8;        // elements that a thread loads together

struct SortArgs {
    const void* ids;
    int n, V, passes, bits;  // bits per pass
    int64_t pad;
    int2* list[2];  // (row, position)
    int* listed;    // numbers of listed chunks, set to 0 here
};

// One cluster sorts (row, position) by row, stably: least significant digit first.
// CTA r owns the r-th run of the list and each of its warps a run of that, so list
// order is (CTA, warp, iteration, lane). Per pass: every warp counts its digits, and
// an element's rank among the equal digits before it in the run falls out of the same
// step (match over the 32 lanes plus the running count); the counts become offsets
// (over warps inside the CTA, over CTAs through distributed shared memory, over
// digits); every element goes to its digit's offset plus its rank. Runs of up to
// 32 * kItems elements stay in registers between the two steps (65536 tokens in all);
// longer ones are read and ranked again.
//
// Bound by latency: 9 us of a pass are four barriers, the remote counts and scattered
// 8-byte stores, which the SMs of the cluster issue one sector per clock. Two passes over
// 65001 tokens: 20 us; one over 16384 ids below 64: 8 us. An earlier version of it decided
// for 16 CTAs (28 us against 41 with 8); 512 threads, as the registers of 1024 spill.
template <int IDT>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortArgs a) {
    __shared__ int count[kSortWarps][kBins];
    __shared__ int total[kBins];   // this CTA's digit counts, read by the whole cluster
    __shared__ int start[kBins];
    __shared__ int warp_sum[kBins / 32];
    launch_dependents();
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks());
    const int rank = static_cast<int>(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int runs = ctas * kSortWarps;
    const int per = ((a.n + runs - 1) / runs + 31) / 32 * 32;  // a warp's run
    const int64_t first = static_cast<int64_t>(rank * kSortWarps + warp) * per;
    const int lo = static_cast<int>(first < a.n ? first : a.n);
    const int hi = static_cast<int>(first + per < a.n ? first + per : a.n);
    const int mask = (1 << a.bits) - 1;
    const bool single = per <= 32 * kItems;
    wait_for_primary();
    if (rank == 0 && threadIdx.x < 2) a.listed[threadIdx.x] = 0;

    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        const int2* in_list = a.list[(pass + 1) & 1];
        int2* out_list = a.list[pass & 1];
        int k[kItems], p[kItems], off[kItems];
        auto load = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                const int i = i0 + 32 * j + lane;
                if (i < hi) {
                    if (pass > 0) {
                        const int2 x = in_list[i];
                        k[j] = x.x;
                        p[j] = x.y;
                    } else {
                        const int v = row_of<IDT>(a.ids, i, a.V, a.pad);
                        k[j] = v < 0 ? a.V : v;
                        p[j] = i;
                    }
                }
            }
        };
        // off = rank among the equal digits that the warp has counted so far
        auto rank_items = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                if (i0 + 32 * j >= hi) break;
                const bool in = i0 + 32 * j + lane < hi;
                const int d = in ? (k[j] >> shift) & mask : kBins;
                const unsigned same = __match_any_sync(0xffffffffu, d);
                const int ahead = __popc(same & ((1u << lane) - 1u));
                if (in) off[j] = count[warp][d] + ahead;
                __syncwarp();
                if (in && ahead == 0) count[warp][d] += __popc(same);
                __syncwarp();
            }
        };
        for (int b = lane; b < kBins; b += 32) count[warp][b] = 0;
        __syncwarp();
        for (int i0 = lo; i0 < hi; i0 += 32 * kItems) {
            load(i0);
            rank_items(i0);
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
            int run = 0;
#pragma unroll 8
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = run;
                run += c;
            }
            total[threadIdx.x] = run;
        }
        cluster.sync();
        if (threadIdx.x < kBins) {
            int c[kSortCluster];  // all remote loads in flight together
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r)
                c[r] = r < ctas ? *cluster.map_shared_rank(&total[threadIdx.x], r) : 0;
            int before = 0, all = 0;
#pragma unroll
            for (int r = 0; r < kSortCluster; ++r) {
                if (r < rank) before += c[r];
                all += c[r];
            }
            int incl = all;  // inclusive scan over the digits
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            if (lane == 31) warp_sum[warp] = incl;
            start[threadIdx.x] = incl - all + before;
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
            int add = 0;
            for (int w = 0; w < warp; ++w) add += warp_sum[w];
            start[threadIdx.x] += add;
        }
        __syncthreads();
        for (int i0 = lo; i0 < hi; i0 += 32 * kItems) {
            if (!single) {
                load(i0);
                rank_items(i0);
            }
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                const int i = i0 + 32 * j + lane;
                if (i < hi) {
                    const int d = (k[j] >> shift) & mask;
                    const int at = start[d] + off[j] + (single ? count[warp][d] : 0);
                    out_list[at] = make_int2(k[j], p[j]);
                }
            }
        }
        // the list of this pass is complete and every CTA has read the others'
        // totals before either is touched again
        cluster.sync();
    }
}

// ---- sums over the segments ------------------------------------------------------
constexpr int kChunk = 32;    // sorted tokens per block
constexpr int kThreads = 256; // columns' threads per block, at most
constexpr int kGroups = 8;    // warps that share a long segment
constexpr int kLong = 16;     // a segment is long when it goes on over so many chunks

struct GradArgs {
    const int2* tok;  // sorted (row, position)
    const float* dm;
    const float* dS;
    int n, V, D;
    float s, s2, inv_cap;
    float* mw;        // update: the table; deltas: Sw only
    float* Sw;
    float* out_m;     // sums and deltas
    float* out_S;
    float* part;      // [chunk][head m, head S, tail m, tail S][D]
    int* listed;      // numbers of short and of long entries
    int4* list;       // (first chunk, last chunk, row) of the segments that cross a border:
                      // short ones from the front, long ones from the back
    int chunks;
};

// The capped update of capped_pair (common.cuh) with the division by the cap as a
// product; a delta that is not a number leaves its parameter as it is, as there.
__device__ __forceinline__ void capped_step(float& m, float& S, float dm, float dS, float inv_cap) {
    const float bound = sqrtf(fmaxf(S, 1e-10f)) * inv_cap;
    m += dm == dm ? fminf(fmaxf(dm, -bound), bound) : 0.f;
    const float raw = S + (dS == dS ? fminf(fmaxf(dS, -bound), bound) : 0.f);
    S = raw <= 0.f ? 1e-5f : raw;
}

// The row's parameters that the final form needs.
template <int VEC, int MODE>
__device__ __forceinline__ void params(const GradArgs& a, int64_t o, float (&mean)[VEC],
                                       float (&w)[VEC]) {
    if (MODE != TAGI_WGRAD_SUMS) ldv<VEC>(a.Sw + o, w);
    if (MODE == TAGI_WGRAD_UPDATE) ldv<VEC>(a.mw + o, mean);
}

// The sums of one row at offset o in their final form.
template <int VEC, int MODE, typename T>
__device__ __forceinline__ void finish(const GradArgs& a, int64_t o, const T (&m)[VEC],
                                       const T (&S)[VEC], float (&mean)[VEC], float (&w)[VEC]) {
    float gm[VEC], gS[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        gm[e] = static_cast<float>(m[e] * a.s);
        gS[e] = static_cast<float>(S[e] * a.s2);
    }
    if (MODE == TAGI_WGRAD_UPDATE) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            capped_step(mean[e], w[e], w[e] * gm[e], w[e] * w[e] * gS[e], a.inv_cap);
        stv<VEC>(a.mw + o, mean);
        stv<VEC>(a.Sw + o, w);
        return;
    }
    if (MODE == TAGI_WGRAD_DELTAS) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            gm[e] *= w[e];
            gS[e] *= w[e] * w[e];
        }
    }
    stv<VEC>(a.out_m + o, gm);
    stv<VEC>(a.out_S + o, gS);
}

// Rows [32 * block * warps, ...) that no token names get zero sums: every lane looks
// its row up in the sorted list, then the warp writes the absent ones.
template <int VEC>
__device__ __forceinline__ void zero_rows(const GradArgs& a, int block) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int64_t v0 = (static_cast<int64_t>(block) * warps + (threadIdx.x >> 5)) * 32;
    const int64_t v = v0 + lane;
    bool absent = false;
    if (v < a.V) {
        int lo = 0, hi = a.n;  // first token whose row is >= v
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.tok[mid].x < v) lo = mid + 1;
            else hi = mid;
        }
        absent = lo == a.n || a.tok[lo].x != v;
    }
    float zero[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
    for (unsigned rows = __ballot_sync(0xffffffffu, absent); rows != 0; rows &= rows - 1) {
        const int64_t o = (v0 + __ffs(rows) - 1) * a.D;
        for (int j = lane * VEC; j < a.D; j += 32 * VEC) {
            stv<VEC>(a.out_m + o + j, zero);
            stv<VEC>(a.out_S + o + j, zero);
        }
    }
}

// What happens to the running sum behind a token.
enum { GOES_ON = 0, FINAL = 1, HEAD = 2, TAIL = 3 };

// AHEAD tokens' delta rows, and the parameters of the rows that end among them, are
// loaded before any of them is added: a row of one token (most rows of a text batch)
// would otherwise wait for its parameters alone.
//
// Bound by HBM: every delta row once, the named rows of the table once each way. Update
// of 50021 x 770 from 65001 tokens: 84 us for 446 MB, 5.3 TB/s (rows of 3080 bytes in
// random order); sums of 16384 x 512: 16 us cold, 4.2 TB/s.
template <int VEC, int MODE>
__global__ void __launch_bounds__(kThreads) reduce_kernel(const GradArgs a) {
    constexpr int AHEAD = 4;  // 8 cost occupancy: 112 us instead of 87 for the update above, then
    __shared__ int4 tok[kChunk];  // row, position, what happens behind it
    launch_dependents();
    wait_for_primary();  // the sorted list
    if (static_cast<int>(blockIdx.x) >= a.chunks) {
        if (blockIdx.y == 0) zero_rows<VEC>(a, blockIdx.x - a.chunks);
        return;
    }
    const int c0 = blockIdx.x * kChunk;
    int cnt = min(kChunk, a.n - c0);
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        static_assert(kChunk == 32, "a lane per token");
        const int t = c0 + lane;
        const int2 x = t < a.n ? a.tok[t] : make_int2(a.V, 0);
        const int prev = c0 > 0 ? a.tok[c0 - 1].x : -1;
        int next = __shfl_down_sync(0xffffffffu, x.x, 1);
        if (lane == 31) next = t + 1 < a.n ? a.tok[t + 1].x : -1;
        const bool ends = next != x.x || lane == 31;
        const bool after = lane == 31 && next == x.x, before = x.x == prev;
        tok[lane] = make_int4(x.x, x.y, !ends ? GOES_ON : (before ? HEAD : (after ? TAIL : FINAL)), 0);
        if (after && !before && x.x < a.V && blockIdx.y == 0) {
            // a segment begins here and goes on: look for its last chunk
            int last = blockIdx.x + 1, hi = a.chunks - 1;
            for (int step = 1; last < hi;) {  // chunk k begins with this row: true up to the last
                const int k = min(last + step, hi);
                if (a.tok[static_cast<int64_t>(k) * kChunk].x == x.x) {
                    last = k;
                    step *= 2;
                } else {
                    hi = k - 1;
                    step = max(1, (hi - last + 1) / 2);
                }
            }
            const bool longer = last - static_cast<int>(blockIdx.x) >= kLong;
            const int at = atomicAdd(&a.listed[longer], 1);
            a.list[longer ? a.chunks - 1 - at : at] = make_int4(blockIdx.x, last, x.x, 0);
        }
    }
    __syncthreads();
    const int j = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    if (j >= a.D) return;
    float m[VEC], S[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.f;
    for (int i0 = 0; i0 < cnt; i0 += AHEAD) {
        if (tok[i0].x >= a.V) break;  // dropped tokens sort last
        float xm[AHEAD][VEC], xS[AHEAD][VEC], mean[AHEAD][VEC], w[AHEAD][VEC];
        int row[AHEAD], kind[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int4 t = tok[i0 + u];
            row[u] = t.x;
            kind[u] = i0 + u < cnt && t.x < a.V ? t.z : -1;
            if (kind[u] >= 0) {
                const int64_t o = static_cast<int64_t>(t.y) * a.D + j;
                ldv_once<VEC>(a.dm + o, xm[u]);
                ldv_once<VEC>(a.dS + o, xS[u]);
            }
            if (kind[u] == FINAL)
                params<VEC, MODE>(a, static_cast<int64_t>(t.x) * a.D + j, mean[u], w[u]);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (kind[u] < 0) break;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                m[e] += xm[u][e];
                S[e] += xS[u][e];
            }
            if (kind[u] == GOES_ON) continue;
            if (kind[u] == FINAL) {
                finish<VEC, MODE>(a, static_cast<int64_t>(row[u]) * a.D + j, m, S, mean[u], w[u]);
            } else {
                float* p = a.part +
                           (static_cast<int64_t>(blockIdx.x) * 4 + (kind[u] == HEAD ? 0 : 2)) * a.D;
                stv<VEC>(p + j, m);
                stv<VEC>(p + a.D + j, S);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.f;
        }
    }
}

// Adds the partials of chunks c, c + step, ... <= last of the segment that begins in
// chunk `begin`, columns j..
template <int VEC>
__device__ __forceinline__ void add_partials(const GradArgs& a, int begin, int c, int step, int last,
                                             int j, double (&m)[VEC], double (&S)[VEC]) {
#pragma unroll 4
    for (int k = c; k <= last; k += step) {
        const float* p = a.part + (static_cast<int64_t>(k) * 4 + (k == begin ? 2 : 0)) * a.D;
        float x[VEC], y[VEC];
        ldv<VEC>(p + j, x);
        ldv<VEC>(p + a.D + j, y);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            m[e] += x[e];
            S[e] += y[e];
        }
    }
}

// Segments that cross a border: the tail of the chunk in which one begins and the heads
// of those that it reaches. A warp takes the columns of a short one; for a long one
// kGroups warps share them, each takes every kGroups-th chunk, and their sums are added
// in order. Bound by latency (list, then partials, then parameters): 12 us for the 1500
// crossing segments of the text batch, 6 us for 64 segments of 8 chunks.
template <int VEC, int MODE>
__global__ void __launch_bounds__(32 * kGroups) join_kernel(const GradArgs a) {
    __shared__ double sum[2][kGroups][32 * VEC];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int j = (blockIdx.y * 32 + lane) * VEC;
    wait_for_primary();  // the partials and the list of segments
    const int shorts = a.listed[0], longs = a.listed[1];
    for (int it = blockIdx.x * kGroups + g; it < shorts && j < a.D; it += gridDim.x * kGroups) {
        const int4 c = a.list[it];
        const int64_t o = static_cast<int64_t>(c.z) * a.D + j;
        double m[VEC] = {}, S[VEC] = {};
        float mean[VEC], w[VEC];
        params<VEC, MODE>(a, o, mean, w);
        add_partials<VEC>(a, c.x, c.x, 1, c.y, j, m, S);
        finish<VEC, MODE>(a, o, m, S, mean, w);
    }
    for (int it = blockIdx.x; it < longs; it += gridDim.x) {
        const int4 c = a.list[a.chunks - 1 - it];
        const int64_t o = static_cast<int64_t>(c.z) * a.D + j;
        double m[VEC] = {}, S[VEC] = {};
        if (j < a.D) add_partials<VEC>(a, c.x, c.x + g, kGroups, c.y, j, m, S);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            sum[0][g][lane * VEC + e] = m[e];
            sum[1][g][lane * VEC + e] = S[e];
        }
        __syncthreads();
        if (g == 0 && j < a.D) {
            float mean[VEC], w[VEC];
            params<VEC, MODE>(a, o, mean, w);
            for (int k = 1; k < kGroups; ++k) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    m[e] += sum[0][k][lane * VEC + e];
                    S[e] += sum[1][k][lane * VEC + e];
                }
            }
            finish<VEC, MODE>(a, o, m, S, mean, w);
        }
        __syncthreads();  // the sums are rewritten for the next segment
    }
}

size_t align_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

size_t list_bytes(int64_t n) { return align_up(static_cast<size_t>(n) * sizeof(int2)); }

size_t grad_ws(int64_t n, int64_t D) {
    if (n <= 0) return 0;
    const size_t chunks = static_cast<size_t>((n + kChunk - 1) / kChunk);
    // the sorted list twice, the list of segments and its lengths, the partial sums
    return 2 * list_bytes(n) + align_up((chunks + 1) * sizeof(int4)) +
           align_up(chunks * 4 * static_cast<size_t>(D) * sizeof(float));
}

// The widest vectors that every row of every operand allows.
int vec_of(int64_t D, uintptr_t bits) {
    if (D % 4 == 0 && (bits & 15) == 0) return 4;
    return D % 2 == 0 && (bits & 7) == 0 ? 2 : 1;
}

uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <int IDT>
int launch_sort(const SortArgs& a, cudaStream_t st, const char* what) {
    // a CTA takes 1024 tokens or more, so that small batches skip the cluster barriers
    int ctas = 1;
    while (ctas < kSortCluster && a.n > ctas * 1024) ctas *= 2;
    // the attribute belongs to the current device's copy of the kernel
    const cudaError_t e =
        cudaFuncSetAttribute(sort_kernel<IDT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: clusters of %d refused (%s)", what, kSortCluster, cudaGetErrorString(e));
        return TAGI_E_LAUNCH;
    }
    launch_early(sort_kernel<IDT>, {dim3(ctas), dim3(kSortThreads), st, 0, dim3(ctas)}, a);
    return check_launch(what);
}

template <int VEC, int MODE>
int launch_grad(GradArgs a, cudaStream_t st, const char* what) {
    // the columns in even slices of whole warps
    const int vecs = (a.D + VEC - 1) / VEC;
    const int slices = (vecs + kThreads - 1) / kThreads;
    const int threads = ((vecs + slices - 1) / slices + 31) / 32 * 32;
    a.chunks = (a.n + kChunk - 1) / kChunk;
    int64_t zero = 0;
    if (MODE != TAGI_WGRAD_UPDATE) zero = (static_cast<int64_t>(a.V) + threads - 1) / threads;
    if (a.chunks + zero == 0) return TAGI_OK;
    TAGI_REQUIRE(a.chunks + zero <= INT32_MAX, TAGI_E_UNSUPPORTED, "%s: sizes beyond the grid", what);
    const dim3 grid(static_cast<unsigned>(a.chunks + zero), slices);
    launch_early(reduce_kernel<VEC, MODE>, {grid, dim3(threads), st}, a);
    const int rc = check_launch(what);
    if (rc || a.chunks <= 1) return rc;
    const int cols = (vecs + 31) / 32;
    const unsigned most = (a.chunks + kGroups - 2) / kGroups;  // a warp per segment
    const unsigned fill = (kNumSMs * 8 + cols - 1) / cols;
    launch_early(join_kernel<VEC, MODE>,
                 {dim3(most < fill ? most : fill, cols), dim3(32 * kGroups), st}, a);
    return check_launch(what);
}

template <int VEC>
int launch_mode(const GradArgs& a, int mode, cudaStream_t st, const char* what) {
    if (mode == TAGI_WGRAD_SUMS) return launch_grad<VEC, TAGI_WGRAD_SUMS>(a, st, what);
    if (mode == TAGI_WGRAD_DELTAS) return launch_grad<VEC, TAGI_WGRAD_DELTAS>(a, st, what);
    return launch_grad<VEC, TAGI_WGRAD_UPDATE>(a, st, what);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int tagi_embedding_lookup(const void* ids, int id_type, const float* mw, const float* Sw,
                                     float* mz, float* Sz, int64_t n, int64_t V, int64_t D,
                                     int64_t padding_idx, double scale, void* stream) {
    const char* what = "tagi_embedding_lookup";
    TAGI_REQUIRE(n >= 0 && V >= 1 && D >= 1 && V < INT32_MAX && D <= INT32_MAX, TAGI_E_BAD_ARG,
                 "%s: bad sizes", what);
    TAGI_REQUIRE(id_type >= ID_F32 && id_type <= ID_I64, TAGI_E_BAD_ARG, "%s: bad id type", what);
    TAGI_REQUIRE(id_type != ID_F32 || V <= (1 << 24), TAGI_E_BAD_ARG,
                 "%s: float ids hold rows below 2^24 only", what);
    if (n == 0) return TAGI_OK;
    TAGI_REQUIRE(ids && mw && Sw && mz && Sz, TAGI_E_BAD_ARG, "%s: null pointer", what);
    const int vec = vec_of(D, bits_of(mw) | bits_of(Sw) | bits_of(mz) | bits_of(Sz));
    // the square is formed before either is rounded: sqrt(512) scales variances by 512
    const float s = static_cast<float>(scale), s2 = static_cast<float>(scale * scale);
    cudaStream_t st = as_stream(stream);
#define LOOKUP(VEC, IDT)                                                                      \
    launch_early(lookup_kernel<VEC, IDT>, {dim3(grid_1d(n * (D / VEC), 256)), dim3(256), st}, \
                 ids, mw, Sw, mz, Sz, n, static_cast<int>(V), static_cast<int>(D),            \
                 padding_idx, s, s2)
#define LOOKUP_V(IDT)                 \
    if (vec == 4) LOOKUP(4, IDT);     \
    else if (vec == 2) LOOKUP(2, IDT); \
    else LOOKUP(1, IDT)
    if (id_type == ID_F32) { LOOKUP_V(ID_F32); }
    else if (id_type == ID_I32) { LOOKUP_V(ID_I32); }
    else { LOOKUP_V(ID_I64); }
#undef LOOKUP_V
#undef LOOKUP
    return check_launch(what);
}

extern "C" size_t tagi_embedding_grad_workspace_size(int64_t n, int64_t D) { return grad_ws(n, D); }

extern "C" int tagi_embedding_grad(const void* ids, int id_type, const float* dmz, const float* dSz,
                                   int64_t n, int64_t V, int64_t D, int64_t padding_idx,
                                   double scale, int mode, float* mw, float* Sw, float* out_m,
                                   float* out_S, float cap_factor, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const char* what = "tagi_embedding_grad";
    TAGI_REQUIRE(n >= 0 && V >= 1 && D >= 1 && n <= (1 << 30) && V < INT32_MAX && D <= (1 << 20),
                 TAGI_E_BAD_ARG, "%s: bad sizes", what);
    TAGI_REQUIRE(id_type >= ID_F32 && id_type <= ID_I64, TAGI_E_BAD_ARG, "%s: bad id type", what);
    TAGI_REQUIRE(id_type != ID_F32 || V <= (1 << 24), TAGI_E_BAD_ARG,
                 "%s: float ids hold rows below 2^24 only", what);
    TAGI_REQUIRE(mode == TAGI_WGRAD_SUMS || mode == TAGI_WGRAD_DELTAS || mode == TAGI_WGRAD_UPDATE,
                 TAGI_E_BAD_ARG, "%s: bad mode", what);
    TAGI_REQUIRE(n == 0 || (ids && dmz && dSz), TAGI_E_BAD_ARG, "%s: null pointer", what);
    if (mode == TAGI_WGRAD_UPDATE)
        TAGI_REQUIRE(mw && Sw && cap_factor > 0.f, TAGI_E_BAD_ARG, "%s: bad update args", what);
    else
        TAGI_REQUIRE(out_m && out_S && (mode == TAGI_WGRAD_SUMS || Sw), TAGI_E_BAD_ARG,
                     "%s: null pointer", what);
    TAGI_REQUIRE(n == 0 || (workspace && workspace_bytes >= grad_ws(n, D)), TAGI_E_WORKSPACE,
                 "%s: needs %zu bytes of workspace", what, grad_ws(n, D));
    TAGI_REQUIRE((bits_of(workspace) & 15) == 0, TAGI_E_ALIGNMENT,
                 "%s: workspace not 16-byte aligned", what);
    TAGI_REQUIRE((D + 31) / 32 <= 65535, TAGI_E_UNSUPPORTED, "%s: sizes beyond the grid", what);
    cudaStream_t st = as_stream(stream);
    GradArgs g{};
    if (n > 0) {
        SortArgs a{};
        char* w = static_cast<char*>(workspace);
        for (int i = 0; i < 2; ++i) a.list[i] = reinterpret_cast<int2*>(w + i * list_bytes(n));
        const size_t chunks = static_cast<size_t>((n + kChunk - 1) / kChunk);
        g.listed = a.listed = reinterpret_cast<int*>(w + 2 * list_bytes(n));
        g.list = reinterpret_cast<int4*>(a.listed) + 1;
        g.part = reinterpret_cast<float*>(w + 2 * list_bytes(n) +
                                          align_up((chunks + 1) * sizeof(int4)));
        a.ids = ids;
        a.n = static_cast<int>(n);
        a.V = static_cast<int>(V);
        a.pad = padding_idx;
        int bits = 1;
        while ((V >> bits) != 0) ++bits;  // rows 0..V, V being the dropped tokens'
        a.passes = (bits + 7) / 8;
        a.bits = (bits + a.passes - 1) / a.passes;
        const int rc = id_type == ID_F32   ? launch_sort<ID_F32>(a, st, what)
                       : id_type == ID_I32 ? launch_sort<ID_I32>(a, st, what)
                                           : launch_sort<ID_I64>(a, st, what);
        if (rc) return rc;
        g.tok = a.list[(a.passes - 1) & 1];
    }
    g.dm = dmz;
    g.dS = dSz;
    g.n = static_cast<int>(n);
    g.V = static_cast<int>(V);
    g.D = static_cast<int>(D);
    g.s = static_cast<float>(scale);
    g.s2 = static_cast<float>(scale * scale);  // as in the lookup
    g.inv_cap = 1.0f / cap_factor;
    g.mw = mw;
    g.Sw = Sw;
    g.out_m = out_m;
    g.out_S = out_S;
    const int vec = vec_of(D, bits_of(dmz) | bits_of(dSz) | bits_of(mw) | bits_of(Sw) |
                                  bits_of(out_m) | bits_of(out_S));
    if (vec == 4) return launch_mode<4>(g, mode, st, what);
    if (vec == 2) return launch_mode<2>(g, mode, st, what);
    return launch_mode<1>(g, mode, st, what);
}
