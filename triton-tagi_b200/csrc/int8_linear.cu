// Mean and variance of a linear layer from 8-bit operands (tcgen05, kind::i8).
//
//   mz[m,n] = a_m[m] b_m[n] sum_k x_m[m,k] w_m[n,k] + mb[n]
//   Sz[m,n] = a_2[m] b_S[n] sum_k x_2[m,k] w_S[n,k]
//           + a_S[m] b_2[n] sum_k x_S[m,k] w_2[n,k] + Sb[n]
//
// x: codes of the tokens' means (signed), squared means and variances (unsigned);
// w: codes of the weights' means, mu^2 + S and variances; a, b: the scales of each
// token and of each output channel. The three products are exact (32-bit sums).
//
// Tiles. The weights are the A operand (128 channels: tensor-memory lanes) and the
// tokens the B operand (BN columns), so a lane is a channel: its scales and bias are
// registers, and for one token a warp stores 32 neighbouring channels of a row of the
// output straight from tensor memory. Few tokens take a narrow B tile (16 columns)
// instead of padding 128 rows. Blocks of grid.z 0 form the variance (two products,
// two accumulators), those of grid.z 1 the mean.
//
// Warp roles: warp 0 issues the tensor-map copies (128 bytes of the reduction of both
// operands per stage, 128-byte swizzle), warp 1 allocates tensor memory and issues
// the MMAs, warps 2-5 read the accumulators (lane quarter w % 4) and store.
//
// Every wait is bounded: on timeout a block records an error word
// (tagi_device_status), stops issuing, lets its own copies and MMAs land and frees
// its tensor memory.
#include <cuda.h>

#include <mutex>

#include "common.cuh"
#include "int8_linear.cuh"
#include "tagi_b200.h"

namespace tagi {

__device__ int g_int8_error = 0;
__device__ unsigned long long g_int8_wait_ns = 2000000000ull;
__device__ int g_int8_force_abort = 0;

namespace {

constexpr unsigned long long kDrainNs = 2000000000ull;
constexpr int kBK = 128;     // bytes of the reduction per stage
constexpr int kThreads = 192;

template <int BN>
struct Plan {
    static constexpr int STAGE = 128 * kBK + BN * kBK;
    static constexpr int STAGES = BN >= 128 ? 3 : (BN >= 64 ? 4 : 5);
    static constexpr int COLS = 2 * BN < 32 ? 32 : 2 * BN;
    static constexpr int SMEM = STAGES * STAGE + 1024;  // 1024: alignment of the swizzled tiles
};

struct Maps {
    CUtensorMap x[3], w[3];  // means, second operand, variances
};

struct Int8Args {
    const float* xs;  // 3 x M: scales of means, x_2, x_S
    const float* ws;  // 3 x N: scales of means, w_2, w_S
    const float* mb;
    const float* Sb;
    float* mz;
    float* Sz;
    int M, N, K;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ unsigned long long globaltimer() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
// False if the block gave up, or if this wait ran out (the block then gives up).
__device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort,
                                            int code) {
    const unsigned long long t0 = globaltimer();
    const unsigned long long limit = *const_cast<volatile unsigned long long*>(&g_int8_wait_ns);
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (*abort) return false;
        if (globaltimer() - t0 > limit) {
            *abort = 1;
            atomicCAS(&g_int8_error, 0, code);
            return false;
        }
    }
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort,
                                          int code) {
    return mbar_try(bar, parity) || mbar_wait_slow(bar, parity, abort, code);
}
// For copies and MMAs in flight, which must land before the block may exit.
__device__ __noinline__ bool mbar_drain(uint64_t* bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try(bar, parity))
        if (globaltimer() - t0 > kDrainNs) return false;
    return true;
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
                 "r"(bytes)
                 : "memory");
}
// Tile copy from this GPU's own memory to this block alone. x is a multiple of kBK
// bytes, so it starts on a 16-byte boundary.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Descriptor of a K-major tile of rows of 128 bytes in 128-byte swizzle: groups of 8
// rows 1024 bytes apart (stride byte offset); bit 46: the descriptor version of
// sm_100; layout type 2: 128-byte swizzle. A step of 32 bytes along the reduction
// inside the swizzle atom adds 2 to the start address field.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: 32-bit integer accumulator, A and B signed or unsigned
// 8-bit, M = 128, N = bn.
__device__ __forceinline__ uint32_t instr_desc(bool sign, int bn) {
    const uint32_t t = sign ? 1u : 0u;
    return (2u << 4) | (t << 7) | (t << 10) | (static_cast<uint32_t>(bn >> 3) << 17) |
           (static_cast<uint32_t>(128 >> 4) << 24);
}

template <int BN>
__global__ void __launch_bounds__(kThreads) int8_linear_kernel(const Int8Args g,
                                                               const __grid_constant__ Maps maps) {
    using P = Plan<BN>;
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t full[P::STAGES], empty[P::STAGES], done;
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    __shared__ float scale[2][BN];
    char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * 128, m0 = blockIdx.y * BN;
    const bool var = blockIdx.z == 0;
    const int kblocks = (g.K + kBK - 1) / kBK;
    const int iters = var ? 2 * kblocks : kblocks;
    volatile int* ab = &abort_flag;

    if (threadIdx.x == 0) {
        for (int s = 0; s < P::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        abort_flag = g_int8_force_abort;
        if (abort_flag) atomicCAS(&g_int8_error, 0, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_base)),
                     "r"(P::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            for (int it = 0; it < iters; ++it) {
                const int s = it % P::STAGES;
                if (*ab) break;
                if (it >= P::STAGES && !mbar_wait(&empty[s], ((it / P::STAGES) - 1) & 1, ab, 11))
                    break;
                const bool second = it >= kblocks;
                const int k = (second ? it - kblocks : it) * kBK;
                // variance: x_2 with w_S, then x_S with w_2; mean: x_m with w_m
                const CUtensorMap* x = &maps.x[var ? (second ? 2 : 1) : 0];
                const CUtensorMap* w = &maps.w[var ? (second ? 1 : 2) : 0];
                const uint32_t dst = smem_u32(smem + s * P::STAGE);
                mbar_expect_tx(&full[s], P::STAGE);
                tma_load(dst, w, k, n0, &full[s]);
                tma_load(dst + 128 * kBK, x, k, m0, &full[s]);
                issued = it + 1;
            }
            // copies still in flight (after an abort) land before the block may exit
            for (int it = issued > P::STAGES ? issued - P::STAGES : 0; it < issued; ++it)
                if (!mbar_drain(&full[it % P::STAGES], (it / P::STAGES) & 1))
                    atomicCAS(&g_int8_error, 0, 13);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = instr_desc(!var, BN);
            for (int it = 0; it < iters; ++it) {
                const int s = it % P::STAGES;
                if (!mbar_wait(&full[s], (it / P::STAGES) & 1, ab, 12)) break;
                tc_fence_after();
                const bool second = it >= kblocks;
                const uint32_t base = smem_u32(smem + s * P::STAGE);
                const uint64_t a = tile_desc(base), b = tile_desc(base + 128 * kBK);
                const uint32_t d = tmem + (second ? BN : 0);
                const bool first = it == 0 || it == kblocks;
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k)
                    mma_i8(d, a + 2 * k, b + 2 * k, idesc, first && k == 0 ? 0u : 1u);
                mma_commit(&empty[s]);
            }
            mma_commit(&done);
        }
    } else {
        const int t = threadIdx.x - 64;
        for (int i = t; i < 2 * BN; i += 128) {
            const int c = i / BN, m = m0 + i % BN;
            const int which = var ? (c == 0 ? 1 : 2) : 0;
            scale[c][i % BN] = m < g.M ? g.xs[static_cast<int64_t>(which) * g.M + m] : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int quarter = warp & 3;
        const int n = n0 + quarter * 32 + lane;
        float b0 = 0.f, b1 = 0.f, bias = 0.f;
        if (n < g.N) {
            b0 = g.ws[(var ? 2 * static_cast<int64_t>(g.N) : 0) + n];
            b1 = var ? g.ws[static_cast<int64_t>(g.N) + n] : 0.f;
            const float* bp = var ? g.Sb : g.mb;
            bias = bp ? bp[n] : 0.f;
        }
        float* out = var ? g.Sz : g.mz;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(&done, 0, ab, 14) && !*ab);
        if (ok) {
            tc_fence_after();
            const uint32_t t0 = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < BN; c += 16) {
                if (m0 + c >= g.M) break;
                uint32_t r0[16], r1[16];
                tmem_ld16(t0 + c, r0);
                if (var) tmem_ld16(t0 + BN + c, r1);
                tmem_wait_ld();
                if (n < g.N) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int m = m0 + c + e;
                        if (m < g.M) {
                            float z = scale[0][c + e] * b0 * static_cast<float>(static_cast<int>(r0[e]));
                            if (var)
                                z += scale[1][c + e] * b1 * static_cast<float>(static_cast<int>(r1[e]));
                            out[static_cast<int64_t>(m) * g.N + n] = z + bias;
                        }
                    }
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        if (lane == 0 && !mbar_drain(&done, 0)) atomicCAS(&g_int8_error, 0, 15);
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(P::COLS));
    }
}

// The driver's tensor-map encoder, looked up through the runtime.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static std::once_flag once;
    static EncodeTiledFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
        cudaGetLastError();
    });
    return fn;
}

// Map of a matrix of codes (rows x K bytes, row stride ld) read in boxes of
// box_rows x 128 bytes; bytes behind K and rows behind the last read as 0.
bool encode(CUtensorMap* map, const void* p, int64_t rows, int64_t K, int64_t ld, int box_rows) {
    const cuuint64_t dim[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
    const cuuint64_t stride[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t es[2] = {1, 1};
    return encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dim, stride,
                          box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
int launch(const Int8Args& g, const Maps& maps, cudaStream_t st, const char* what) {
    using P = Plan<BN>;
    // the attribute belongs to the current device's copy of the kernel
    const cudaError_t e = cudaFuncSetAttribute(
        int8_linear_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, P::SMEM);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: cannot reserve %d bytes of shared memory (%s)", what, P::SMEM,
                  cudaGetErrorString(e));
        return TAGI_E_LAUNCH;
    }
    const int64_t my = (static_cast<int64_t>(g.M) + BN - 1) / BN;
    TAGI_REQUIRE(my <= 65535, TAGI_E_UNSUPPORTED, "%s: too many rows", what);
    const dim3 grid((g.N + 127) / 128, static_cast<unsigned>(my), 2);
    int8_linear_kernel<BN><<<grid, kThreads, P::SMEM, st>>>(g, maps);
    count_tc_launch();
    return check_launch(what);
}

}  // namespace

int int8_device_status(int reset) {
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int));
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("tagi_device_status: %s", cudaGetErrorString(e));
        return TAGI_E_LAUNCH;
    }
    if (reset && v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(int));
    }
    return v;
}

cudaError_t int8_set_wait_limit(unsigned long long ns, int force) {
    const cudaError_t e = cudaMemcpyToSymbol(g_int8_wait_ns, &ns, sizeof(ns));
    return e != cudaSuccess ? e : cudaMemcpyToSymbol(g_int8_force_abort, &force, sizeof(force));
}

}  // namespace tagi

using namespace tagi;

extern "C" int tagi_int8_moment_matmul(const int8_t* x_m, const uint8_t* x_2, const uint8_t* x_S,
                                       const float* x_scales, int64_t ldx, const int8_t* w_m,
                                       const uint8_t* w_2, const uint8_t* w_S,
                                       const float* w_scales, int64_t ldw, const float* mb,
                                       const float* Sb, float* mz, float* Sz, int64_t M, int64_t N,
                                       int64_t K, void* stream) {
    const char* what = "tagi_int8_moment_matmul";
    // 255 * 255 * K stays below 2^31
    TAGI_REQUIRE(M >= 0 && N >= 0 && K >= 1 && M <= INT32_MAX && N <= INT32_MAX && K <= 33025,
                 TAGI_E_BAD_ARG, "%s: bad sizes (the reduction may have 1 to 33025 terms)", what);
    if (M == 0 || N == 0) return TAGI_OK;
    TAGI_REQUIRE(x_m && x_2 && x_S && x_scales && w_m && w_2 && w_S && w_scales && mz && Sz,
                 TAGI_E_BAD_ARG, "%s: null pointer", what);
    TAGI_REQUIRE(ldx >= K && ldw >= K, TAGI_E_BAD_ARG, "%s: rows overlap", what);
    uintptr_t bits = static_cast<uintptr_t>(ldx) | static_cast<uintptr_t>(ldw);
    for (const void* p : {static_cast<const void*>(x_m), static_cast<const void*>(x_2),
                          static_cast<const void*>(x_S), static_cast<const void*>(w_m),
                          static_cast<const void*>(w_2), static_cast<const void*>(w_S)})
        bits |= reinterpret_cast<uintptr_t>(p);
    TAGI_REQUIRE((bits & 15) == 0, TAGI_E_ALIGNMENT,
                 "%s: rows of codes must start on 16-byte boundaries", what);
    TAGI_REQUIRE(encode_tiled() != nullptr, TAGI_E_LAUNCH, "%s: no tensor-map encoder", what);
    const int bn = M <= 16 ? 16 : (M <= 64 ? 64 : 128);
    Maps maps;
    const void* x[3] = {x_m, x_2, x_S};
    const void* w[3] = {w_m, w_2, w_S};
    for (int i = 0; i < 3; ++i)
        TAGI_REQUIRE(encode(&maps.x[i], x[i], M, K, ldx, bn) && encode(&maps.w[i], w[i], N, K, ldw, 128),
                     TAGI_E_LAUNCH, "%s: the tensor maps were refused", what);
    const Int8Args g{x_scales, w_scales, mb, Sb, mz, Sz, static_cast<int>(M), static_cast<int>(N),
                     static_cast<int>(K)};
    cudaStream_t st = as_stream(stream);
    if (bn == 16) return launch<16>(g, maps, st, what);
    if (bn == 64) return launch<64>(g, maps, st, what);
    return launch<128>(g, maps, st, what);
}
