// Residual addition and RMSNorm of Gaussian rows, with the output in 32 bits or in
// 8 bits with scales, and its backward pass; and rows put into 8 bits on their own.
//
//   h_m = a_m + r_m,  h_S = a_S + r_S                       (the residual stream)
//   inv = 1 / sqrt(mean(h_m^2 + h_S) + eps)
//   mz  = inv h_m w,  Sz = inv^2 (h_S (w^2 + Sw) + Sw h_m^2)
//
// 8 bits. With p = h_m w and t = h_S (w^2 + Sw) + Sw h_m^2, and P, T the row's
// largest |p| and t rounded to fp32, a row is held as
//   q_m = rint(127 p / P)      scale inv P / 127        (signed)
//   q_2 = rint(255 (p / P)^2)  scale (inv P)^2 / 255    (unsigned: mz^2)
//   q_S = rint(255 t / T)      scale inv^2 T / 255      (unsigned)
// inv cancels in the codes, so they do not depend on the order in which the row was
// summed. They are decided in double: a code is the nearest to the exact quotient,
// whatever kernel variant formed it.
//
// A row that holds a value that is not finite has codes 0 and scales NaN, so that
// what is computed from it is NaN; a row of zeros has codes 0 and scales 0.

#include <cstdint>

#include "common.cuh"
#include "tagi_b200.h"

namespace tagi {
namespace {

// What a row kernel writes.
enum { OUT_F32 = 0, OUT_INT8 = 1, OUT_QUANT = 2, OUT_QUANT_W = 3 };

struct NormArgs {
    const float* am;
    const float* aS;
    const float* rm;  // null: no residual
    const float* rS;
    const float* w;
    const float* Sw;
    float* hm;  // null without a residual
    float* hS;
    float* mz;
    float* Sz;
    float* inv;
    int8_t* qm;
    uint8_t* q2;
    uint8_t* qS;
    float* scales;  // 3 x rows
    int64_t ldq, rows;
    int ni;
    float eps;
};

template <int VEC>
__device__ __forceinline__ void ld(const float* p, float (&v)[VEC]) {
    if (VEC == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x;
        v[1 % VEC] = x.y;
        v[2 % VEC] = x.z;
        v[3 % VEC] = x.w;
    } else {
        v[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void st(float* p, const float (&v)[VEC]) {
    if (VEC == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1 % VEC], v[2 % VEC], v[3 % VEC]);
    else
        *p = v[0];
}
template <int VEC, typename T>
__device__ __forceinline__ void st8(T* p, const int (&v)[VEC]) {
    if (VEC == 4) {
        const uint32_t x = (v[0] & 255) | (v[1 % VEC] & 255) << 8 | (v[2 % VEC] & 255) << 16 |
                           static_cast<uint32_t>(v[3 % VEC] & 255) << 24;
        *reinterpret_cast<uint32_t*>(p) = x;
    } else {
        *p = static_cast<T>(v[0]);
    }
}

// Magnitude of x as an ordered key: infinities and NaN above every finite value.
__device__ __forceinline__ unsigned mag(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr unsigned kInfBits = 0x7f800000u;
// The same for a value that counts from 0 up: a finite one below 0 is 0.
__device__ __forceinline__ unsigned mag_pos(float x) {
    const unsigned m = mag(x);
    return x < 0.f && m < kInfBits ? 0u : m;
}

// What a row is reduced to: sum of m^2 + S, largest |p|, t and (weights) u as keys. One
// barrier for all of them, and sums in a fixed order.
struct RowStats {
    float sum;
    unsigned P, T, U;
};
template <int OUT, int WARPS>
__device__ __forceinline__ void reduce_row(RowStats& r, RowStats* red) {
    constexpr bool NORM = OUT == OUT_F32 || OUT == OUT_INT8, CODES = OUT != OUT_F32;
    if (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
    }
    if (CODES) {
        r.P = __reduce_max_sync(0xffffffffu, r.P);
        r.T = __reduce_max_sync(0xffffffffu, r.T);
        if (OUT == OUT_QUANT_W) r.U = __reduce_max_sync(0xffffffffu, r.U);
    }
    if (WARPS == 1) return;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = r;
    __syncthreads();
    r = red[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) {
        const RowStats o = red[i];
        r.sum += o.sum;
        r.P = max(r.P, o.P);
        r.T = max(r.T, o.T);
        r.U = max(r.U, o.U);
    }
}

// p, t and (weights) u = m^2 + S of one element, in double: products of two fp32
// values are exact there.
template <int OUT>
struct Elem {
    double p, t, u;
    __device__ __forceinline__ Elem(float m, float S, float w, float Sw) {
        const double dm = m, dS = S;
        if (OUT == OUT_INT8) {
            const double dw = w, ds = Sw;
            p = dm * dw;
            t = fma(ds, dm * dm, dS * fma(dw, dw, ds));
            u = 0.0;
        } else {
            p = dm;
            t = dS;
            u = OUT == OUT_QUANT_W ? fma(dm, dm, dS) : 0.0;
        }
    }
};

struct RowScales {
    double p, t, u;     // largest magnitudes
    double ip, it, iu;  // and their reciprocals (0 for a row of zeros)
    float sm, s2, sS;
};

// x / d from the reciprocal of d, with one correction step: exact quotients come
// out exact, so ties between two codes fall as the division would let them.
__device__ __forceinline__ double quotient(double x, double d, double inv) {
    const double q = x * inv;
    return fma(fma(-q, d, x), inv, q);
}

// Scales of a row from its largest magnitudes.
template <int OUT>
__device__ __forceinline__ RowScales row_scales(unsigned P, unsigned T, unsigned U, float inv) {
    RowScales r;
    const float nan = __uint_as_float(0x7fffffffu);
    if (P >= kInfBits || T >= kInfBits || U >= kInfBits) {
        r.p = r.t = r.u = r.ip = r.it = r.iu = 0.0;
        r.sm = r.s2 = r.sS = nan;
        return r;
    }
    const float p = __uint_as_float(P), t = __uint_as_float(T), u = __uint_as_float(U);
    r.p = p;
    r.t = t;
    r.u = u;
    r.ip = p > 0.f ? 1.0 / r.p : 0.0;
    r.it = t > 0.f ? 1.0 / r.t : 0.0;
    r.iu = u > 0.f ? 1.0 / r.u : 0.0;
    const float a = inv * p;
    r.sm = a / 127.f;
    r.s2 = OUT == OUT_QUANT_W ? u / 255.f : a * a / 255.f;
    r.sS = inv * inv * t / 255.f;
    return r;
}

// Codes of one element.
template <int OUT>
__device__ __forceinline__ void codes(const Elem<OUT>& e, const RowScales& r, int& qm, int& q2,
                                      int& qS) {
    const double x = quotient(e.p, r.p, r.ip);
    qm = __double2int_rn(127.0 * x);
    q2 = OUT == OUT_QUANT_W ? __double2int_rn(255.0 * fmax(quotient(e.u, r.u, r.iu), 0.0))
                            : __double2int_rn(255.0 * x * x);
    qS = __double2int_rn(255.0 * fmax(quotient(e.t, r.t, r.it), 0.0));
    // P is rounded: the largest element itself may come out a hair above the top code
    qm = max(-127, min(127, qm));
    q2 = min(255, q2);
    qS = min(255, qS);
}

// One row per group of WARPS warps, its stream held in registers: thread i of the
// group has vectors i, i + 32 WARPS, ... (NV at most). One pass over the inputs.
//
// Bound by HBM: 32 bytes per element (27 with codes). 8192 x 4096: 163 us, 6.6 TB/s, the
// rate of a copy; 16384 x 512 with codes: 42 us, 5.4 TB/s. Forming the quotients of the
// codes in fp32 and only those near the middle of two in double took as long (44 us):
// the double arithmetic hides behind the loads. 777 x 1001, one element per load: 11 us,
// bound by latency.
template <int OUT, int VEC, int WARPS, int NV>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS) row_kernel(const NormArgs g) {
    __shared__ RowStats red[WARPS];
    launch_dependents();
    wait_for_primary();
    constexpr int T = 32 * WARPS;
    const int64_t row = WARPS == 1
                            ? blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5)
                            : blockIdx.x;
    if (row >= g.rows) return;
    const int i0 = (WARPS == 1 ? threadIdx.x & 31 : threadIdx.x) * VEC;
    const int64_t base = row * g.ni;
    constexpr bool NORM = OUT == OUT_F32 || OUT == OUT_INT8;
    float m[NV][VEC], S[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = i0 + k * T * VEC;
        if (j < g.ni) {
            ld<VEC>(g.am + base + j, m[k]);
            ld<VEC>(g.aS + base + j, S[k]);
        }
    }
    if (NORM && g.rm) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = i0 + k * T * VEC;
            if (j < g.ni) {
                float x[VEC], y[VEC];
                ld<VEC>(g.rm + base + j, x);
                ld<VEC>(g.rS + base + j, y);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    m[k][e] += x[e];
                    S[k][e] += y[e];
                }
                st<VEC>(g.hm + base + j, m[k]);
                st<VEC>(g.hS + base + j, S[k]);
            }
        }
    }
    RowStats rs{0.f, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = i0 + k * T * VEC;
        if (j < g.ni) {
            float w[VEC] = {}, sw[VEC] = {};
            if (OUT == OUT_INT8) {
                ld<VEC>(g.w + j, w);
                ld<VEC>(g.Sw + j, sw);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (NORM) rs.sum += fmaf(m[k][e], m[k][e], S[k][e]);
                if (OUT != OUT_F32) {
                    const Elem<OUT> el(m[k][e], S[k][e], w[e], sw[e]);
                    rs.P = max(rs.P, mag(static_cast<float>(el.p)));
                    rs.T = max(rs.T, mag_pos(static_cast<float>(el.t)));
                    if (OUT == OUT_QUANT_W) rs.U = max(rs.U, mag_pos(static_cast<float>(el.u)));
                }
            }
        }
    }
    reduce_row<OUT, WARPS>(rs, red);
    float inv = 1.f;
    if (NORM) {
        inv = 1.0f / sqrtf(rs.sum / static_cast<float>(g.ni) + g.eps);
        if (i0 == 0 && g.inv) g.inv[row] = inv;
    }
    if (OUT == OUT_F32) {
        const float inv2 = inv * inv;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = i0 + k * T * VEC;
            if (j < g.ni) {
                float w[VEC], sw[VEC];
                ld<VEC>(g.w + j, w);
                ld<VEC>(g.Sw + j, sw);
                float z[VEC], v[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float x = m[k][e];
                    z[e] = inv * x * w[e];
                    v[e] = inv2 * (S[k][e] * (w[e] * w[e] + sw[e]) + sw[e] * x * x);
                }
                st<VEC>(g.mz + base + j, z);
                st<VEC>(g.Sz + base + j, v);
            }
        }
        return;
    }
    const RowScales r = row_scales<OUT>(rs.P, rs.T, rs.U, inv);
    if (i0 == 0) {
        g.scales[row] = r.sm;
        g.scales[g.rows + row] = r.s2;
        g.scales[2 * g.rows + row] = r.sS;
    }
    const bool bad = rs.P >= kInfBits || rs.T >= kInfBits || rs.U >= kInfBits;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = i0 + k * T * VEC;
        if (j < g.ni) {
            float w[VEC] = {}, sw[VEC] = {};
            if (OUT == OUT_INT8) {
                ld<VEC>(g.w + j, w);
                ld<VEC>(g.Sw + j, sw);
            }
            int a[VEC], b[VEC], c[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const Elem<OUT> el(m[k][e], S[k][e], w[e], sw[e]);
                codes<OUT>(el, r, a[e], b[e], c[e]);
                if (bad) a[e] = b[e] = c[e] = 0;
            }
            const int64_t o = row * g.ldq + j;
            st8<VEC>(g.qm + o, a);
            st8<VEC>(g.q2 + o, b);
            st8<VEC>(g.qS + o, c);
        }
    }
}

// Rows too long for registers: one block per row, the stream read again for every
// pass (from h where a residual was added, from the input where not).
template <int OUT>
__global__ void __launch_bounds__(512) long_row_kernel(const NormArgs g) {
    constexpr int WARPS = 16;
    __shared__ RowStats red[WARPS];
    launch_dependents();
    wait_for_primary();
    constexpr bool NORM = OUT == OUT_F32 || OUT == OUT_INT8;
    const int64_t row = blockIdx.x;
    const int64_t base = row * g.ni;
    const bool add = NORM && g.rm;
    const float* hm = (add ? g.hm : g.am) + base;
    const float* hS = (add ? g.hS : g.aS) + base;
    RowStats rs{0.f, 0u, 0u, 0u};
    for (int j = threadIdx.x; j < g.ni; j += blockDim.x) {
        float x = g.am[base + j], y = g.aS[base + j];
        if (add) {
            x += g.rm[base + j];
            y += g.rS[base + j];
            g.hm[base + j] = x;
            g.hS[base + j] = y;
        }
        if (NORM) rs.sum += fmaf(x, x, y);
        if (OUT != OUT_F32) {
            const Elem<OUT> el(x, y, OUT == OUT_INT8 ? g.w[j] : 0.f, OUT == OUT_INT8 ? g.Sw[j] : 0.f);
            rs.P = max(rs.P, mag(static_cast<float>(el.p)));
            rs.T = max(rs.T, mag_pos(static_cast<float>(el.t)));
            if (OUT == OUT_QUANT_W) rs.U = max(rs.U, mag_pos(static_cast<float>(el.u)));
        }
    }
    reduce_row<OUT, WARPS>(rs, red);
    float inv = 1.f;
    if (NORM) {
        inv = 1.0f / sqrtf(rs.sum / static_cast<float>(g.ni) + g.eps);
        if (threadIdx.x == 0 && g.inv) g.inv[row] = inv;
    }
    // every thread reads back the elements that it wrote itself
    if (OUT == OUT_F32) {
        for (int j = threadIdx.x; j < g.ni; j += blockDim.x) {
            const float x = hm[j], w = g.w[j], sw = g.Sw[j];
            g.mz[base + j] = inv * x * w;
            g.Sz[base + j] = inv * inv * (hS[j] * (w * w + sw) + sw * x * x);
        }
        return;
    }
    const RowScales r = row_scales<OUT>(rs.P, rs.T, rs.U, inv);
    if (threadIdx.x == 0) {
        g.scales[row] = r.sm;
        g.scales[g.rows + row] = r.s2;
        g.scales[2 * g.rows + row] = r.sS;
    }
    const bool bad = rs.P >= kInfBits || rs.T >= kInfBits || rs.U >= kInfBits;
    for (int j = threadIdx.x; j < g.ni; j += blockDim.x) {
        const Elem<OUT> el(hm[j], hS[j], OUT == OUT_INT8 ? g.w[j] : 0.f,
                           OUT == OUT_INT8 ? g.Sw[j] : 0.f);
        int a, b, c;
        codes<OUT>(el, r, a, b, c);
        const int64_t o = row * g.ldq + j;
        g.qm[o] = static_cast<int8_t>(bad ? 0 : a);
        g.q2[o] = static_cast<uint8_t>(bad ? 0 : b);
        g.qS[o] = static_cast<uint8_t>(bad ? 0 : c);
    }
}

template <int OUT, int VEC, int WARPS, int NV>
int launch_row(const NormArgs& g, cudaStream_t st, const char* what) {
    const int threads = WARPS == 1 ? 128 : 32 * WARPS;
    const int64_t blocks = WARPS == 1 ? (g.rows + 3) / 4 : g.rows;
    TAGI_REQUIRE(blocks <= INT32_MAX, TAGI_E_UNSUPPORTED, "%s: too many rows", what);
    launch_early(row_kernel<OUT, VEC, WARPS, NV>,
                 {dim3(static_cast<unsigned>(blocks)), dim3(threads), st}, g);
    return check_launch(what);
}

template <int OUT, int VEC>
int launch_width(const NormArgs& g, cudaStream_t st, const char* what) {
    const int vecs = (g.ni + VEC - 1) / VEC;
    if (vecs <= 64) return launch_row<OUT, VEC, 1, 2>(g, st, what);
    if (vecs <= 128) return launch_row<OUT, VEC, 1, 4>(g, st, what);
    if (vecs <= 256) return launch_row<OUT, VEC, 2, 4>(g, st, what);
    if (vecs <= 512) return launch_row<OUT, VEC, 4, 4>(g, st, what);
    if (vecs <= 1024) return launch_row<OUT, VEC, 8, 4>(g, st, what);
    if (vecs <= 2048) return launch_row<OUT, VEC, 16, 4>(g, st, what);
    TAGI_REQUIRE(g.rows <= INT32_MAX, TAGI_E_UNSUPPORTED, "%s: too many rows", what);
    launch_early(long_row_kernel<OUT>, {dim3(static_cast<unsigned>(g.rows)), dim3(512), st}, g);
    return check_launch(what);
}

template <int OUT>
int launch_norm(const NormArgs& g, cudaStream_t st, const char* what) {
    uintptr_t bits = 0;
    for (const void* p : {static_cast<const void*>(g.am), static_cast<const void*>(g.aS),
                          static_cast<const void*>(g.rm), static_cast<const void*>(g.rS),
                          static_cast<const void*>(g.w), static_cast<const void*>(g.Sw),
                          static_cast<const void*>(g.hm), static_cast<const void*>(g.hS),
                          static_cast<const void*>(g.mz), static_cast<const void*>(g.Sz)})
        bits |= reinterpret_cast<uintptr_t>(p);
    uintptr_t bits8 = static_cast<uintptr_t>(g.ldq);
    for (const void* p : {static_cast<const void*>(g.qm), static_cast<const void*>(g.q2),
                          static_cast<const void*>(g.qS)})
        bits8 |= reinterpret_cast<uintptr_t>(p);
    if (g.ni % 4 == 0 && (bits & 15) == 0 && (bits8 & 3) == 0)
        return launch_width<OUT, 4>(g, st, what);
    return launch_width<OUT, 1>(g, st, what);
}

// code * scale of one of the three operands (blockIdx.y), VEC codes per thread; the
// block's y rows at a time. Bound by HBM: 16384 x 512 in 25 us, 6.0 TB/s.
template <int VEC>
__global__ void values_kernel(const NormArgs g, float* vm, float* v2, float* vS) {
    launch_dependents();
    wait_for_primary();
    const int which = blockIdx.y;
    const uint8_t* q = which == 0 ? reinterpret_cast<const uint8_t*>(g.qm)
                                  : (which == 1 ? g.q2 : g.qS);
    float* v = which == 0 ? vm : (which == 1 ? v2 : vS);
    const float* sc = g.scales + which * g.rows;
    for (int64_t r = blockIdx.x * static_cast<int64_t>(blockDim.y) + threadIdx.y; r < g.rows;
         r += static_cast<int64_t>(gridDim.x) * blockDim.y) {
        const float s = sc[r];
#pragma unroll 4
        for (int j = threadIdx.x * VEC; j < g.ni; j += blockDim.x * VEC) {
            const uint8_t* p = q + r * g.ldq + j;
            const uint32_t x = VEC == 4 ? *reinterpret_cast<const uint32_t*>(p) : *p;
            float out[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const uint32_t b = (x >> (8 * e)) & 255u;
                out[e] = s * (which == 0 ? static_cast<float>(static_cast<int8_t>(b))
                                         : static_cast<float>(b));
            }
            st<VEC>(v + r * g.ni + j, out);
        }
    }
}

// ---- backward -------------------------------------------------------------------
//   d_m = r_m + (inv w) dz_m,  d_S = r_S + (inv w)^2 dz_S
//   sums over rows: g_m = sum inv h dz_m,  g_S = sum (inv h)^2 dz_S
// Both are formed in one pass: block (slice, columns) walks its rows with its columns'
// sums in registers, kBackThreads / x rows at a time (x threads along the columns), adds
// the groups' sums in order and leaves them in the workspace; a second launch adds the
// slices in order and applies them (a single slice applies its own). Bound by HBM: 28 bytes per element. 16384 x 512:
// 43.6 us with the second launch, 5.4 TB/s; without the row groups there were four times
// the slices and the second launch alone took 15 us.
constexpr int kBackThreads = 512;
constexpr int kBackCols = 128;  // threads along the columns, at most

// What becomes of gamma's sums.
struct GammaOut {
    int mode;
    double* sums;
    float* w;
    float* Sw;
    float* d_w;
    float* d_Sw;
    float cap;
};
__device__ __forceinline__ void gamma_out(const GammaOut& o, int j, int ni, double a, double b) {
    if (o.mode == TAGI_WGRAD_SUMS) {
        o.sums[j] = a;
        o.sums[ni + j] = b;
        return;
    }
    const float S = o.Sw[j];
    const float dm = static_cast<float>(a) * S, dS = static_cast<float>(b) * S * S;
    if (o.mode == TAGI_WGRAD_DELTAS) {
        o.d_w[j] = dm;
        o.d_Sw[j] = dS;
        return;
    }
    float m = o.w[j], v = S;
    capped_pair(m, v, dm, dS, o.cap);
    o.w[j] = m;
    o.Sw[j] = v;
}

struct BackArgs {
    GammaOut gamma;  // used here when one slice holds all rows
    const float* dm;
    const float* dS;
    const float* h;
    const float* inv;
    const float* w;
    const float* rm;  // null: no deltas of the stream
    const float* rS;
    float* om;
    float* oS;
    double* part;  // [slice][2][ni]
    int64_t rows;
    int ni, slice_rows;
};

template <int VEC>
__global__ void __launch_bounds__(kBackThreads) back_kernel(const BackArgs g) {
    __shared__ double red[2][kBackThreads * VEC];
    launch_dependents();
    wait_for_primary();
    const int j = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    const int groups = blockDim.y, grp = threadIdx.y;
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * g.slice_rows;
    const int64_t r1 = r0 + g.slice_rows < g.rows ? r0 + g.slice_rows : g.rows;
    double sm[VEC], sS[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sm[e] = sS[e] = 0.0;
    if (j < g.ni) {
        float w[VEC];
        ld<VEC>(g.w + j, w);
#pragma unroll 2
        for (int64_t r = r0 + grp; r < r1; r += groups) {
            const int64_t o = r * g.ni + j;
            const float inv = g.inv[r];
            float dm[VEC], dS[VEC], h[VEC], xm[VEC], xS[VEC];
            ld<VEC>(g.dm + o, dm);
            ld<VEC>(g.dS + o, dS);
            ld<VEC>(g.h + o, h);
            if (g.rm) {
                ld<VEC>(g.rm + o, xm);
                ld<VEC>(g.rS + o, xS);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) xm[e] = xS[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float t = inv * w[e], x = inv * h[e];
                xm[e] += t * dm[e];
                xS[e] += t * t * dS[e];
                sm[e] += static_cast<double>(x * dm[e]);
                sS[e] += static_cast<double>(x * x * dS[e]);
            }
            st<VEC>(g.om + o, xm);
            st<VEC>(g.oS + o, xS);
        }
    }
    const int at = (grp * blockDim.x + threadIdx.x) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        red[0][at + e] = sm[e];
        red[1][at + e] = sS[e];
    }
    __syncthreads();
    // a thread per column
    const int cols = blockDim.x * VEC;
    for (int c = grp * blockDim.x + threadIdx.x; c < cols; c += kBackThreads) {
        const int col = blockIdx.y * cols + c;
        if (col >= g.ni) continue;
        double a = red[0][c], b = red[1][c];
        for (int k = 1; k < groups; ++k) {
            a += red[0][k * cols + c];
            b += red[1][k * cols + c];
        }
        if (gridDim.x == 1) {
            gamma_out(g.gamma, col, g.ni, a, b);
            continue;
        }
        double* p = g.part + static_cast<int64_t>(blockIdx.x) * 2 * g.ni + col;
        p[0] = a;
        p[g.ni] = b;
    }
}

// Adds the slices' sums: 8 columns per block, 32 threads per column, each every 32nd
// slice (a fixed order), their sums by a shuffle tree of fixed shape.
__global__ void __launch_bounds__(256) back_finish_kernel(const double* part, int slices, int ni,
                                                          const GammaOut out) {
    __shared__ double red[2][8][33];
    const int c = threadIdx.x & 7, g = threadIdx.x >> 3;
    const int col = blockIdx.x * 8 + c;
    double a = 0.0, b = 0.0;
    wait_for_primary();  // the slices' sums
    if (col < ni) {
#pragma unroll 8
        for (int s = g; s < slices; s += 32) {
            a += part[static_cast<int64_t>(s) * 2 * ni + col];
            b += part[static_cast<int64_t>(s) * 2 * ni + ni + col];
        }
    }
    red[0][c][g] = a;
    red[1][c][g] = b;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;  // a warp per column
    a = red[0][warp][lane];
    b = red[1][warp][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    const int j = blockIdx.x * 8 + warp;
    if (lane == 0 && j < ni) gamma_out(out, j, ni, a, b);
}

// Threads along the columns of `vecs` vectors, and slices of rows: two blocks per SM (what
// the registers allow: 512 threads of 64), 2 rows or more for each of a block's groups.
int back_x(int64_t vecs) {
    int x = 32;
    while (x < kBackCols && x < vecs) x *= 2;
    return x;
}
int slices_of(int64_t rows, int64_t ni, int vec) {
    const int64_t vecs = (ni + vec - 1) / vec;
    const int x = back_x(vecs);
    const int64_t cols = (vecs + x - 1) / x;
    int64_t s = (kNumSMs * 2 + cols - 1) / cols;
    const int64_t per = 2 * (kBackThreads / x);
    const int64_t most = (rows + per - 1) / per;
    if (s > most) s = most;
    return static_cast<int>(s < 1 ? 1 : s);
}

}  // namespace
}  // namespace tagi

using namespace tagi;

#define ROWS_CHECK()                                                                        \
    TAGI_REQUIRE(rows >= 0 && ni >= 1 && ni <= (1 << 24), TAGI_E_BAD_ARG, "%s: bad sizes", what)

extern "C" int tagi_add_rmsnorm_forward(const float* ma, const float* Sa, const float* mr,
                                        const float* Sr, const float* mw, const float* Sw,
                                        float* hm, float* hS, float* mz, float* Sz,
                                        float* inv_rms, int64_t rows, int64_t ni, float eps,
                                        void* stream) {
    const char* what = "tagi_add_rmsnorm_forward";
    ROWS_CHECK();
    if (rows == 0) return TAGI_OK;
    TAGI_REQUIRE(ma && Sa && mw && Sw && mz && Sz && inv_rms, TAGI_E_BAD_ARG, "%s: null pointer",
                 what);
    TAGI_REQUIRE((mr == nullptr) == (Sr == nullptr) && (!mr || (hm && hS)), TAGI_E_BAD_ARG,
                 "%s: a residual needs mean, variance and both stream outputs", what);
    NormArgs g{};
    g.am = ma; g.aS = Sa; g.rm = mr; g.rS = Sr; g.w = mw; g.Sw = Sw;
    g.hm = mr ? hm : nullptr; g.hS = mr ? hS : nullptr;
    g.mz = mz; g.Sz = Sz; g.inv = inv_rms;
    g.rows = rows; g.ni = static_cast<int>(ni); g.eps = eps;
    return launch_norm<OUT_F32>(g, as_stream(stream), what);
}

extern "C" int tagi_add_rmsnorm_int8(const float* ma, const float* Sa, const float* mr,
                                     const float* Sr, const float* mw, const float* Sw, float* hm,
                                     float* hS, int8_t* q_m, uint8_t* q_2, uint8_t* q_S,
                                     float* scales, int64_t ldq, int64_t rows, int64_t ni,
                                     float eps, void* stream) {
    const char* what = "tagi_add_rmsnorm_int8";
    ROWS_CHECK();
    if (rows == 0) return TAGI_OK;
    TAGI_REQUIRE(ma && Sa && mw && Sw && q_m && q_2 && q_S && scales, TAGI_E_BAD_ARG,
                 "%s: null pointer", what);
    TAGI_REQUIRE((mr == nullptr) == (Sr == nullptr) && (!mr || (hm && hS)), TAGI_E_BAD_ARG,
                 "%s: a residual needs mean, variance and both stream outputs", what);
    TAGI_REQUIRE(ldq >= ni, TAGI_E_BAD_ARG, "%s: rows of codes overlap", what);
    NormArgs g{};
    g.am = ma; g.aS = Sa; g.rm = mr; g.rS = Sr; g.w = mw; g.Sw = Sw;
    g.hm = mr ? hm : nullptr; g.hS = mr ? hS : nullptr;
    g.qm = q_m; g.q2 = q_2; g.qS = q_S; g.scales = scales; g.ldq = ldq;
    g.rows = rows; g.ni = static_cast<int>(ni); g.eps = eps;
    return launch_norm<OUT_INT8>(g, as_stream(stream), what);
}

extern "C" int tagi_quantize_moments(const float* m, const float* S, int weights, int8_t* q_m,
                                     uint8_t* q_2, uint8_t* q_S, float* scales, int64_t ldq,
                                     int64_t rows, int64_t ni, void* stream) {
    const char* what = "tagi_quantize_moments";
    ROWS_CHECK();
    if (rows == 0) return TAGI_OK;
    TAGI_REQUIRE(m && S && q_m && q_2 && q_S && scales, TAGI_E_BAD_ARG, "%s: null pointer", what);
    TAGI_REQUIRE(ldq >= ni, TAGI_E_BAD_ARG, "%s: rows of codes overlap", what);
    NormArgs g{};
    g.am = m; g.aS = S; g.qm = q_m; g.q2 = q_2; g.qS = q_S; g.scales = scales; g.ldq = ldq;
    g.rows = rows; g.ni = static_cast<int>(ni);
    return weights ? launch_norm<OUT_QUANT_W>(g, as_stream(stream), what)
                   : launch_norm<OUT_QUANT>(g, as_stream(stream), what);
}

extern "C" int tagi_int8_values(const int8_t* q_m, const uint8_t* q_2, const uint8_t* q_S,
                                const float* scales, int64_t ldq, float* v_m, float* v_2,
                                float* v_S, int64_t rows, int64_t ni, void* stream) {
    const char* what = "tagi_int8_values";
    ROWS_CHECK();
    if (rows == 0) return TAGI_OK;
    TAGI_REQUIRE(q_m && q_2 && q_S && scales && v_m && v_2 && v_S, TAGI_E_BAD_ARG,
                 "%s: null pointer", what);
    TAGI_REQUIRE(ldq >= ni, TAGI_E_BAD_ARG, "%s: rows of codes overlap", what);
    NormArgs g{};
    g.qm = const_cast<int8_t*>(q_m); g.q2 = const_cast<uint8_t*>(q_2);
    g.qS = const_cast<uint8_t*>(q_S); g.scales = const_cast<float*>(scales);
    g.ldq = ldq; g.rows = rows; g.ni = static_cast<int>(ni);
    uintptr_t bits = static_cast<uintptr_t>(ldq) * 4;  // codes on 4 bytes, values on 16
    for (const void* p : {static_cast<const void*>(v_m), static_cast<const void*>(v_2),
                          static_cast<const void*>(v_S)})
        bits |= reinterpret_cast<uintptr_t>(p);
    for (const void* p : {static_cast<const void*>(q_m), static_cast<const void*>(q_2),
                          static_cast<const void*>(q_S)})
        bits |= reinterpret_cast<uintptr_t>(p) * 4;
    const bool v4 = ni % 4 == 0 && (bits & 15) == 0;
    const int64_t vecs = v4 ? ni / 4 : ni;
    int x = 32;
    while (x < 256 && x < vecs) x *= 2;
    const dim3 block(x, 256 / x), grid(grid_1d(rows, 256 / x, kNumSMs * 32), 3);
    if (v4)
        launch_early(values_kernel<4>, {grid, block, as_stream(stream)}, g, v_m, v_2, v_S);
    else
        launch_early(values_kernel<1>, {grid, block, as_stream(stream)}, g, v_m, v_2, v_S);
    return check_launch(what);
}

extern "C" size_t tagi_add_rmsnorm_backward_workspace_size(int64_t rows, int64_t ni) {
    if (rows < 0 || ni < 1) return 0;
    // the larger of both vector widths: alignment is not known here
    const int a = slices_of(rows, ni, 4), b = slices_of(rows, ni, 1);
    return static_cast<size_t>(a > b ? a : b) * 2 * static_cast<size_t>(ni) * sizeof(double);
}

extern "C" int tagi_add_rmsnorm_backward(const float* dmz, const float* dSz, const float* hm,
                                         const float* inv_rms, const float* rm, const float* rS,
                                         float* d_m, float* d_S, int mode, double* sums, float* mw,
                                         float* Sw, float* d_mw, float* d_Sw, float cap_factor,
                                         int64_t rows, int64_t ni, void* workspace,
                                         size_t workspace_bytes, void* stream) {
    const char* what = "tagi_add_rmsnorm_backward";
    ROWS_CHECK();
    TAGI_REQUIRE(mw && (rows == 0 || (dmz && dSz && hm && inv_rms && d_m && d_S)), TAGI_E_BAD_ARG,
                 "%s: null pointer", what);
    TAGI_REQUIRE((rm == nullptr) == (rS == nullptr), TAGI_E_BAD_ARG,
                 "%s: the stream's deltas need mean and variance", what);
    TAGI_REQUIRE((mode == TAGI_WGRAD_SUMS && sums) ||
                     (mode == TAGI_WGRAD_DELTAS && Sw && d_mw && d_Sw) ||
                     (mode == TAGI_WGRAD_UPDATE && Sw && cap_factor > 0.f),
                 TAGI_E_BAD_ARG, "%s: bad mode or its arguments missing", what);
    const size_t need = tagi_add_rmsnorm_backward_workspace_size(rows, ni);
    TAGI_REQUIRE(workspace && workspace_bytes >= need, TAGI_E_WORKSPACE,
                 "%s: needs %zu bytes of workspace", what, need);
    TAGI_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, TAGI_E_ALIGNMENT,
                 "%s: workspace not 16-byte aligned", what);
    cudaStream_t st = as_stream(stream);
    BackArgs g{};
    g.dm = dmz; g.dS = dSz; g.h = hm; g.inv = inv_rms; g.w = mw; g.rm = rm; g.rS = rS;
    g.om = d_m; g.oS = d_S; g.part = static_cast<double*>(workspace);
    g.gamma = {mode, sums, mw, Sw, d_mw, d_Sw, cap_factor};
    g.rows = rows; g.ni = static_cast<int>(ni);
    uintptr_t bits = 0;
    for (const void* p : {static_cast<const void*>(dmz), static_cast<const void*>(dSz),
                          static_cast<const void*>(hm), static_cast<const void*>(rm),
                          static_cast<const void*>(rS), static_cast<const void*>(mw),
                          static_cast<const void*>(d_m), static_cast<const void*>(d_S)})
        bits |= reinterpret_cast<uintptr_t>(p);
    const bool v4 = ni % 4 == 0 && (bits & 15) == 0;
    const int slices = slices_of(rows, ni, v4 ? 4 : 1);
    const int64_t per = (rows + slices - 1) / slices;
    TAGI_REQUIRE(per <= INT32_MAX, TAGI_E_UNSUPPORTED, "%s: too many rows", what);
    g.slice_rows = static_cast<int>(per < 1 ? 1 : per);
    const int64_t vecs = v4 ? ni / 4 : ni;
    const int x = back_x(vecs);
    const dim3 grid(slices, static_cast<unsigned>((vecs + x - 1) / x)), block(x, kBackThreads / x);
    TAGI_REQUIRE((vecs + x - 1) / x <= 65535, TAGI_E_UNSUPPORTED, "%s: too many columns", what);
    if (v4)
        launch_early(back_kernel<4>, {grid, block, st}, g);
    else
        launch_early(back_kernel<1>, {grid, block, st}, g);
    const int rc = check_launch(what);
    if (rc || slices == 1) return rc;
    launch_early(back_finish_kernel, {dim3(static_cast<unsigned>((ni + 7) / 8)), dim3(256), st},
                 static_cast<const double*>(g.part), slices, g.ni, g.gamma);
    return check_launch(what);
}
