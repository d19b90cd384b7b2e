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
//           it began here and goes on).
//   join    1 launch.  The block of a chunk with a tail adds the heads that follow.
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
    const typename Vec<VEC>::type x = __ldg(reinterpret_cast<const typename Vec<VEC>::type*>(p));
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

template <int VEC, int IDT>
__global__ void lookup_kernel(const void* ids, const float* mw, const float* Sw, float* mz,
                              float* Sz, int64_t n, int V, int D, int64_t pad, float s, float s2) {
    const int per = D / VEC;
    const int64_t total = n * per;
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
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kBins = 256;
constexpr int kSortCluster = 8;  // the largest portable cluster

struct SortArgs {
    const void* ids;
    int n, V, passes, bits;  // bits per pass
    int64_t pad;
    int* key[2];
    int* pos[2];
};

// One cluster sorts (row, position) by row, stably: least significant digit first.
// CTA r owns the r-th run of the list and each of its warps a run of that, so list
// order is (CTA, warp, iteration, lane). Per pass: every warp counts its digits;
// the counts become offsets (over warps inside the CTA, over CTAs through
// distributed shared memory, over digits); every warp walks its run again and puts
// each element at its digit's offset plus its rank among the equal digits of its
// 32 lanes.
template <int IDT>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortArgs a) {
    __shared__ int count[kSortWarps][kBins];
    __shared__ int total[kBins];   // this CTA's digit counts, read by the whole cluster
    __shared__ int start[kBins];
    __shared__ int warp_sum[kBins / 32];
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

    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        const int* key = a.key[(pass + 1) & 1];
        const int* pos = a.pos[(pass + 1) & 1];
        int* key_out = a.key[pass & 1];
        int* pos_out = a.pos[pass & 1];
        auto key_at = [&](int i) {
            if (pass > 0) return key[i];
            const int v = row_of<IDT>(a.ids, i, a.V, a.pad);
            return v < 0 ? a.V : v;
        };
        for (int b = lane; b < kBins; b += 32) count[warp][b] = 0;
        __syncwarp();
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            const int d = i < hi ? (key_at(i) >> shift) & mask : kBins;
            const unsigned same = __match_any_sync(0xffffffffu, d);
            if (d < kBins && (same & ((1u << lane) - 1u)) == 0) count[warp][d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if (threadIdx.x < kBins) {
            int run = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = count[w][threadIdx.x];
                count[w][threadIdx.x] = run;
                run += c;
            }
            total[threadIdx.x] = run;
        }
        cluster.sync();
        if (threadIdx.x < kBins) {
            int before = 0, all = 0;
            for (int r = 0; r < ctas; ++r) {
                const int c = *cluster.map_shared_rank(&total[threadIdx.x], r);
                if (r < rank) before += c;
                all += c;
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
            int add = start[threadIdx.x];
            for (int w = 0; w < warp; ++w) add += warp_sum[w];
            for (int w = 0; w < kSortWarps; ++w) count[w][threadIdx.x] += add;
        }
        __syncthreads();
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const int i = i0 + lane;
            int k = 0, d = kBins;
            if (i < hi) {
                k = key_at(i);
                d = (k >> shift) & mask;
            }
            const unsigned same = __match_any_sync(0xffffffffu, d);
            const int ahead = __popc(same & ((1u << lane) - 1u));
            if (i < hi) {
                const int at = count[warp][d] + ahead;
                key_out[at] = k;
                pos_out[at] = pass > 0 ? pos[i] : i;
            }
            __syncwarp();
            if (i < hi && ahead == 0) count[warp][d] += __popc(same);
            __syncwarp();
        }
        // the list of this pass is complete and every CTA has read the others'
        // totals before either is touched again
        cluster.sync();
    }
}

// ---- sums over the segments ------------------------------------------------------
constexpr int kChunk = 32;    // sorted tokens per block
constexpr int kAhead = 8;     // delta rows loaded ahead of the adds
constexpr int kThreads = 128;

struct GradArgs {
    const int* key;
    const int* pos;
    const float* dm;
    const float* dS;
    int n, V, D, mode;
    float s, s2, cap;
    float* mw;        // update: the table; deltas: Sw only
    float* Sw;
    float* out_m;     // sums and deltas
    float* out_S;
    float* part;      // [chunk][head m, head S, tail m, tail S][D]
};

// The sums of one row's columns j..j+VEC-1 in their final form.
template <int VEC, typename T>
__device__ __forceinline__ void finish(const GradArgs& a, int v, int j, const T (&m)[VEC],
                                       const T (&S)[VEC]) {
    const int64_t o = static_cast<int64_t>(v) * a.D + j;
    float gm[VEC], gS[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        gm[e] = static_cast<float>(m[e] * a.s);
        gS[e] = static_cast<float>(S[e] * a.s2);
    }
    if (a.mode != TAGI_WGRAD_SUMS) {
        float w[VEC];
        ldv<VEC>(a.Sw + o, w);
        if (a.mode == TAGI_WGRAD_UPDATE) {
            float mean[VEC];
            ldv<VEC>(a.mw + o, mean);
#pragma unroll
            for (int e = 0; e < VEC; ++e) capped_pair(mean[e], w[e], w[e] * gm[e], w[e] * w[e] * gS[e], a.cap);
            stv<VEC>(a.mw + o, mean);
            stv<VEC>(a.Sw + o, w);
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            gm[e] *= w[e];
            gS[e] *= w[e] * w[e];
        }
    }
    stv<VEC>(a.out_m + o, gm);
    stv<VEC>(a.out_S + o, gS);
}

template <int VEC>
__global__ void __launch_bounds__(kThreads) reduce_kernel(const GradArgs a) {
    __shared__ int key[kChunk + 2];  // with the neighbours on both sides (-1: none)
    __shared__ int pos[kChunk];
    const int c0 = blockIdx.x * kChunk;
    const int cnt = min(kChunk, a.n - c0);
    for (int i = threadIdx.x; i < cnt + 2; i += kThreads) {
        const int t = c0 + i - 1;
        key[i] = t >= 0 && t < a.n ? a.key[t] : -1;
        if (i >= 1 && i <= cnt) pos[i - 1] = a.pos[t];
    }
    __syncthreads();
    const int j = (blockIdx.y * kThreads + threadIdx.x) * VEC;
    if (j >= a.D || key[1] == a.V) return;  // dropped tokens sort last
    float m[VEC], S[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.f;
    int seg = 0;  // first token of the running segment
    for (int i0 = 0; i0 < cnt; i0 += kAhead) {
        float xm[kAhead][VEC], xS[kAhead][VEC];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u < cnt && key[i0 + u + 1] < a.V) {
                const int64_t o = static_cast<int64_t>(pos[i0 + u]) * a.D + j;
                ldv<VEC>(a.dm + o, xm[u]);
                ldv<VEC>(a.dS + o, xS[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            if (i >= cnt || key[i + 1] >= a.V) break;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                m[e] += xm[u][e];
                S[e] += xS[u][e];
            }
            const int v = key[i + 1];
            const bool last = i == cnt - 1;
            if (!last && key[i + 2] == v) continue;
            const bool before = seg == 0 && key[0] == v, after = last && key[i + 2] == v;
            if (!before && !after) {
                finish<VEC>(a, v, j, m, S);
            } else {
                float* p = a.part + (static_cast<int64_t>(blockIdx.x) * 4 + (before ? 0 : 2)) * a.D;
                stv<VEC>(p + j, m);
                stv<VEC>(p + a.D + j, S);
            }
            seg = i + 1;
#pragma unroll
            for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.f;
        }
    }
}

// Block (c, slice): if a segment begins in chunk c and goes on behind it, the sum
// of its tail and of the heads of the chunks that it reaches. kGroups threads share
// a column, each takes every kGroups-th chunk, and their sums are added in order.
constexpr int kGroups = 8;
template <int VEC>
__global__ void __launch_bounds__(32 * kGroups) join_kernel(const GradArgs a) {
    __shared__ double sum[2][kGroups][32 * VEC];
    const int c = blockIdx.x;
    const int end = (c + 1) * kChunk;
    if (end >= a.n) return;
    const int v = a.key[end - 1];
    if (v == a.V || a.key[end] != v) return;
    const int c0 = c * kChunk;
    if (c0 > 0 && a.key[c0] == v && a.key[c0 - 1] == v) return;  // began in an earlier chunk
    int last = c + 1;  // the last chunk that the segment reaches
    {
        int lo = c + 1, hi = (a.n - 1) / kChunk;
        while (lo < hi) {  // chunk k begins with v: true up to the last
            const int mid = (lo + hi + 1) / 2;
            if (a.key[mid * kChunk] == v) lo = mid;
            else hi = mid - 1;
        }
        last = lo;
    }
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int j = (blockIdx.y * 32 + lane) * VEC;
    double m[VEC], S[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) m[e] = S[e] = 0.0;
    if (j < a.D) {
#pragma unroll 4
        for (int k = c + g; k <= last; k += kGroups) {
            const float* p = a.part + (static_cast<int64_t>(k) * 4 + (k == c ? 2 : 0)) * a.D;
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
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        sum[0][g][lane * VEC + e] = m[e];
        sum[1][g][lane * VEC + e] = S[e];
    }
    __syncthreads();
    if (g != 0 || j >= a.D) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        for (int k = 1; k < kGroups; ++k) {
            m[e] += sum[0][k][lane * VEC + e];
            S[e] += sum[1][k][lane * VEC + e];
        }
    }
    finish<VEC>(a, v, j, m, S);
}

// Rows that no token names get zero sums: one warp per row looks it up in the
// sorted list.
template <int VEC>
__global__ void absent_rows_kernel(const GradArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5;
    float zero[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
    for (int64_t v = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5; v < a.V;
         v += warps) {
        int lo = 0, hi = a.n;  // first token whose row is >= v
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.key[mid] < v) lo = mid + 1;
            else hi = mid;
        }
        if (lo < a.n && a.key[lo] == v) continue;
        for (int j = lane * VEC; j < a.D; j += 32 * VEC) {
            stv<VEC>(a.out_m + v * a.D + j, zero);
            stv<VEC>(a.out_S + v * a.D + j, zero);
        }
    }
}

size_t align_up(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

size_t list_bytes(int64_t n) { return align_up(static_cast<size_t>(n) * 4); }

size_t grad_ws(int64_t n, int64_t D) {
    if (n <= 0) return 0;
    const size_t chunks = static_cast<size_t>((n + kChunk - 1) / kChunk);
    return 4 * list_bytes(n) + align_up(chunks * 4 * static_cast<size_t>(D) * sizeof(float));
}

// The widest vectors that every row of every operand allows.
int vec_of(int64_t D, uintptr_t bits) {
    if (D % 4 == 0 && (bits & 15) == 0) return 4;
    return D % 2 == 0 && (bits & 7) == 0 ? 2 : 1;
}

uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }

template <int IDT>
int launch_sort(const SortArgs& a, cudaStream_t st, const char* what) {
    // a CTA takes 2048 tokens or more, so that small batches skip the cluster barriers
    int ctas = 1;
    while (ctas < kSortCluster && a.n > ctas * 2048) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kSortThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, sort_kernel<IDT>, a);
    return check_launch(what);
}

template <int VEC>
int launch_grad(const GradArgs& a, cudaStream_t st, const char* what) {
    int rc;
    if (a.mode != TAGI_WGRAD_UPDATE) {
        absent_rows_kernel<VEC><<<grid_1d(static_cast<int64_t>(a.V) * 32, 256), 256, 0, st>>>(a);
        if ((rc = check_launch(what))) return rc;
    }
    if (a.n == 0) return TAGI_OK;
    const unsigned chunks = static_cast<unsigned>((a.n + kChunk - 1) / kChunk);
    const int per = kThreads * VEC;
    reduce_kernel<VEC><<<dim3(chunks, (a.D + per - 1) / per), kThreads, 0, st>>>(a);
    if ((rc = check_launch(what))) return rc;
    if (chunks == 1) return TAGI_OK;
    const int jper = 32 * VEC;
    join_kernel<VEC><<<dim3(chunks - 1, (a.D + jper - 1) / jper), 32 * kGroups, 0, st>>>(a);
    return check_launch(what);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

extern "C" int tagi_embedding_lookup(const void* ids, int id_type, const float* mw, const float* Sw,
                                     float* mz, float* Sz, int64_t n, int64_t V, int64_t D,
                                     int64_t padding_idx, float scale, void* stream) {
    const char* what = "tagi_embedding_lookup";
    TAGI_REQUIRE(n >= 0 && V >= 1 && D >= 1 && V < INT32_MAX && D <= INT32_MAX, TAGI_E_BAD_ARG,
                 "%s: bad sizes", what);
    TAGI_REQUIRE(id_type >= ID_F32 && id_type <= ID_I64, TAGI_E_BAD_ARG, "%s: bad id type", what);
    TAGI_REQUIRE(id_type != ID_F32 || V <= (1 << 24), TAGI_E_BAD_ARG,
                 "%s: float ids hold rows below 2^24 only", what);
    if (n == 0) return TAGI_OK;
    TAGI_REQUIRE(ids && mw && Sw && mz && Sz, TAGI_E_BAD_ARG, "%s: null pointer", what);
    const int vec = vec_of(D, bits_of(mw) | bits_of(Sw) | bits_of(mz) | bits_of(Sz));
    const float s2 = scale * scale;
    cudaStream_t st = as_stream(stream);
#define LOOKUP(VEC, IDT)                                                                      \
    lookup_kernel<VEC, IDT><<<grid_1d(n * (D / VEC), 256), 256, 0, st>>>(                     \
        ids, mw, Sw, mz, Sz, n, static_cast<int>(V), static_cast<int>(D), padding_idx, scale, s2)
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
                                   float scale, int mode, float* mw, float* Sw, float* out_m,
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
        for (int i = 0; i < 2; ++i) {
            a.key[i] = reinterpret_cast<int*>(w + (2 * i) * list_bytes(n));
            a.pos[i] = reinterpret_cast<int*>(w + (2 * i + 1) * list_bytes(n));
        }
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
        g.key = a.key[(a.passes - 1) & 1];
        g.pos = a.pos[(a.passes - 1) & 1];
        g.part = reinterpret_cast<float*>(w + 4 * list_bytes(n));
    }
    g.dm = dmz;
    g.dS = dSz;
    g.n = static_cast<int>(n);
    g.V = static_cast<int>(V);
    g.D = static_cast<int>(D);
    g.mode = mode;
    g.s = scale;
    g.s2 = scale * scale;
    g.cap = cap_factor;
    g.mw = mw;
    g.Sw = Sw;
    g.out_m = out_m;
    g.out_S = out_S;
    const int vec = vec_of(D, bits_of(dmz) | bits_of(dSz) | bits_of(mw) | bits_of(Sw) |
                                  bits_of(out_m) | bits_of(out_S));
    if (vec == 4) return launch_grad<4>(g, st, what);
    if (vec == 2) return launch_grad<2>(g, st, what);
    return launch_grad<1>(g, st, what);
}
