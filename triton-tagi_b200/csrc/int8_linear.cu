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
// The weights are the A operand (tensor-memory lanes are channels) and the tokens the
// B operand (columns), so a lane keeps its channel's scales and bias in registers, and
// for one token a warp stores 32 neighbouring channels of a row of the output straight
// from tensor memory. Two kernels:
//
// pair kernel, for many tokens. A cluster of two CTAs computes 256 channels x 256
// tokens with 2-SM MMAs: each CTA stages its 128 channels and half of the tokens, 64
// bytes per clock of the tensor pipe's peak and SM, which the L2 delivers (a single-CTA
// 128 x 128 tile stages 128). Persistent, one pair per two SMs. The
// three products of a tile follow one another through two accumulators of 256 columns:
// the epilogue warps read one while the MMAs fill the other. The first product of the
// variance waits in their registers for the second.
//   8192 x 4096 x 4096: 316 to 350 us per call, one after another under the power cap. A
//   launch alone takes 257 us, 3.2 POP/s: the tensor pipe is active 84 % of the cycles at
//   the 1.6 GHz that its power leaves.
//   16384 x 512 x 2048: 75 to 80 us per call, 67.5 alone. Bound by the epilogue, 12 thousand
//   clocks a tile against 6 of MMAs: 37 us without it, 57 with all of it but the stores.
//
// split kernel, for few tokens or few tiles. 128 channels x BN tokens (16 or 32);
// the (product, reduction block) list of a tile is shared out over a cluster of up to
// 8 CTAs, which exchange their integer sums through distributed shared memory (exact in
// any order).
//   In a captured graph, over weights that are not in the L2: 16 x 4096 x 4096 13 us, 64
//   tokens 16, 128 tokens 23, 256 tokens 36, against 7.7 us for the 50 MB of weights: every
//   16 or 32 tokens read them from the L2 again. 3 x 2048 x 512: 6 us of latency (set-up and
//   first tile 2 us, the others 2, exchange and stores 2), 14.6 us with the call.
//
// Warp roles: warp 0 issues the tensor-map copies (128 bytes of the reduction of both
// operands per stage, 128-byte swizzle), warp 1 allocates tensor memory and issues the
// MMAs (in a pair's first CTA, which a warp of both tells of the stages that have landed),
// the others read the accumulators (lane quarter w % 4) and store.
//
// Every wait is bounded: on timeout a CTA records an error word (tagi_device_status),
// tells its peer, stops issuing, lets its own copies and MMAs land and frees its tensor
// memory.
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
// Scopes of a wait: CTA for arrivals of this CTA's threads, copies and MMAs; CLUSTER where
// the other CTA's threads arrive (arrive_landed, arrive_read).
enum { CTA = 0, CLUSTER = 1 };
template <int SCOPE = CTA>
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    if (SCOPE == CLUSTER)
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, "
            "[%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
            : "memory");
    return ok != 0;
}
struct Abort {
    volatile int* flag;  // this CTA's abort word
    uint32_t peer;       // cluster address of the peer CTA's (0: none)
};
// False if the CTA gave up, or if this wait ran out (it and its peer then give up).
template <int SCOPE>
__device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, const Abort& ab,
                                            int code) {
    const unsigned long long t0 = globaltimer();
    const unsigned long long limit = *const_cast<volatile unsigned long long*>(&g_int8_wait_ns);
    for (;;) {
        if (mbar_try<SCOPE>(bar, parity)) return true;
        if (*ab.flag) return false;
        if (globaltimer() - t0 > limit) {
            *ab.flag = 1;
            if (ab.peer)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ab.peer), "r"(1) : "memory");
            atomicCAS(&g_int8_error, 0, code);
            return false;
        }
    }
}
template <int SCOPE = CTA>
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, const Abort& ab,
                                          int code) {
    return mbar_try<SCOPE>(bar, parity) || mbar_wait_slow<SCOPE>(bar, parity, ab, code);
}
// The same for a whole warp, so that what follows stays uniform.
template <int SCOPE = CTA>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Abort& ab,
                                          int code) {
    return __all_sync(0xffffffffu, mbar_wait<SCOPE>(bar, parity, ab, code));
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}"
        : "=r"(p));
    return p != 0;
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
// Arrive on a barrier given by its cluster address (own or peer CTA). Two kinds, for what
// the other CTA's multiplying warp does behind its wait (an acquire at cluster scope):
//   landed  publishes what this warp has seen: a stage that has landed in this CTA's shared
//           memory, which the MMAs of the pair's first CTA read. The release covers shared
//           memory alone: one of all memory waits for the CTA's output stores, for every
//           stage (8192 x 4096 x 4096: 760 us instead of 273).
//   read    tells that an accumulator has been read. The reads are tensor-memory ones,
//           complete (tcgen05.wait::ld) and ordered by the tcgen05 fences on both sides;
//           nothing else is handed over.
__device__ __forceinline__ void arrive_landed(uint32_t addr) {
    asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory");
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
                 : "memory");
}
__device__ __forceinline__ void arrive_read(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
                 : "memory");
}
// Address of the same shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::
                     : "memory");
}
// A word of another CTA's shared memory, or 0 without reading; no branch, so that many
// are in flight together.
__device__ __forceinline__ int ld_cluster(uint32_t addr, bool read) {
    int v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.s32 %0, 0;\n\t"
        "@p ld.shared::cluster.s32 %0, [%1];\n\t}"
        : "=r"(v)
        : "r"(addr), "r"(read ? 1 : 0)
        : "memory");
    return v;
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
// Asynchronous copy of one word to shared memory, or a 0 without reading.
__device__ __forceinline__ void copy4(float* dst, const float* src, bool read) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(read ? 4 : 0)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on `bar` once all MMAs that this thread issued have completed.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
            smem_u32(bar))
        : "memory");
}
// The same for the pair's MMAs, on the barrier of both CTAs.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_u32(bar)),
        "h"(static_cast<unsigned short>(3))
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
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7])
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
// 8-bit, M = m, N = bn.
__device__ __forceinline__ uint32_t instr_desc(bool sign, int m, int bn) {
    const uint32_t t = sign ? 1u : 0u;
    return (2u << 4) | (t << 7) | (t << 10) | (static_cast<uint32_t>(bn >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// Position in a ring of stages, and the parity of the use of the stage before this one.
template <int STAGES>
struct Ring {
    int s = 0;
    uint32_t parity = 0;  // of this use; the use before has the other
    bool again = false;   // the stage has been used before
    __device__ __forceinline__ void next() {
        if (++s == STAGES) {
            s = 0;
            parity ^= 1u;
            again = true;
        }
    }
};

// Products in their order: variance x_2 w_S, variance x_S w_2, mean x_m w_m; the index
// of the operands and scales (0 means, 1 second operand, 2 variances).
__device__ __forceinline__ int x_of(int product) { return product == 0 ? 1 : (product == 1 ? 2 : 0); }
__device__ __forceinline__ int w_of(int product) { return product == 0 ? 2 : (product == 1 ? 1 : 0); }

// ---- many tokens: CTA pairs, persistent ---------------------------------------------
constexpr int kPairStages = 6;
constexpr int kPairStage = 2 * 128 * kBK;  // 128 channels and 128 tokens per CTA
constexpr int kPairSmem = kPairStages * kPairStage + 1024;
constexpr int kPairReaders = 16;  // epilogue warps: 4 per lane quarter, 64 columns each
constexpr int kTeller = 2 + kPairReaders;  // the warp that tells the leader of landed stages
constexpr int kPairThreads = 32 * (kTeller + 1);

__global__ void __launch_bounds__(kPairThreads, 1)
    int8_pair_kernel(const Int8Args g, const __grid_constant__ Maps maps) {
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t landed[kPairStages], ready[kPairStages],
        empty[kPairStages], acc_full[2], acc_empty[2], done;
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    __shared__ __align__(16) float scale[2][3][256];  // the tile's tokens, by product
    __shared__ float chan[2][5][128];                 // this CTA's channels: by product, Sb, mb
    char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int kblocks = (g.K + kBK - 1) / kBK;
    const int ctiles = (g.N + 255) / 256;
    const int tiles = ctiles * ((g.M + 255) / 256);
    const int pairs = gridDim.x / 2;
    const Abort ab{&abort_flag, map_to(smem_u32(&abort_flag), rank ^ 1)};

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&landed[s], 1);
            mbar_init(&ready[s], 2);  // leader: the stage has landed in both CTAs
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 2 * kPairReaders);  // the epilogue warps of both CTAs
        }
        mbar_init(&done, 1);
        abort_flag = g_int8_force_abort;
        if (abort_flag) atomicCAS(&g_int8_error, 0, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        launch_dependents();  // behind the allocation: see launch_early
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before any remote arrival
    tc_fence_after();
    wait_for_primary();
    const uint32_t tmem = tmem_base;

    // The copying and the multiplying warp run their loops whole and one elected lane
    // issues: with warp-uniform operands a stage of four MMAs costs its issuer 390 clocks,
    // less than the 512 that they take; from a loop of one lane it cost 700, and
    // 8192 x 4096 x 4096 took 297 us instead of 257.
    if (warp == 0) {
        const bool lead = elect_one();
        Ring<kPairStages> ring;
        int it = 0;
        bool alive = true;
        for (int tile = blockIdx.x / 2; tile < tiles && alive; tile += pairs) {
            const int n = (tile % ctiles) * 256 + static_cast<int>(rank) * 128;
            const int m = (tile / ctiles) * 256 + static_cast<int>(rank) * 128;
#pragma unroll 1
            for (int p = 0; p < 3 && alive; ++p) {
                const CUtensorMap* x = &maps.x[x_of(p)];
                const CUtensorMap* w = &maps.w[w_of(p)];
#pragma unroll 1
                for (int k = 0; k < kblocks; ++k, ++it, ring.next()) {
                    alive = ring.again ? warp_wait(&empty[ring.s], ring.parity ^ 1u, ab, 21)
                                       : __all_sync(0xffffffffu, *ab.flag == 0);
                    if (!alive) break;
                    if (lead) {
                        uint64_t* bar = &landed[ring.s];
                        const uint32_t dst = smem_u32(smem + ring.s * kPairStage);
                        mbar_expect_tx(bar, kPairStage);
                        tma_load(dst, w, k * kBK, n, bar);
                        tma_load(dst + 128 * kBK, x, k * kBK, m, bar);
                    }
                    __syncwarp();
                }
            }
        }
        // copies still in flight (after an abort) land before the CTA may exit
        for (int i = it > kPairStages ? it - kPairStages : 0; i < it; ++i)
            if (!mbar_drain(&landed[i % kPairStages], (i / kPairStages) & 1) && lane == 0)
                atomicCAS(&g_int8_error, 0, 23);
    } else if (warp == kTeller) {
        // one barrier for the multiplying warp to wait on instead of one per CTA
        const int my_tiles = (tiles - static_cast<int>(blockIdx.x / 2) + pairs - 1) / pairs;
        const int iters = my_tiles * 3 * kblocks;
        const uint32_t to = map_to(smem_u32(&ready[0]), 0);
        Ring<kPairStages> ring;
#pragma unroll 1
        for (int it = 0; it < iters; ++it, ring.next()) {
            if (!warp_wait(&landed[ring.s], ring.parity, ab, 22)) break;
            if (lane == 0) arrive_landed(to + ring.s * 8);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const bool lead = elect_one();
            Ring<kPairStages> ring;
            int unit = 0;
            bool alive = true;
            for (int tile = blockIdx.x / 2; tile < tiles && alive; tile += pairs) {
#pragma unroll 1
                for (int p = 0; p < 3 && alive; ++p, ++unit) {
                    const uint32_t idesc = instr_desc(p == 2, 256, 256);
                    const int slot = unit & 1;
                    if (unit >= 2 &&
                        !warp_wait<CLUSTER>(&acc_empty[slot], ((unit / 2) - 1) & 1, ab, 24)) {
                        alive = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem + slot * 256;
#pragma unroll 1
                    for (int k = 0; k < kblocks; ++k, ring.next()) {
                        alive = warp_wait<CLUSTER>(&ready[ring.s], ring.parity, ab, 25);
                        if (!alive) break;
                        tc_fence_after();
                        const uint32_t base = smem_u32(smem + ring.s * kPairStage);
                        const uint64_t a = tile_desc(base), b = tile_desc(base + 128 * kBK);
                        if (lead) {
                            mma_i8<true>(d, a, b, idesc, k == 0 ? 0u : 1u);
#pragma unroll
                            for (int j = 1; j < kBK / 32; ++j)
                                mma_i8<true>(d, a + 2 * j, b + 2 * j, idesc, 1u);
                            mma_commit_pair(&empty[ring.s]);
                        }
                        __syncwarp();
                    }
                    if (alive && lead) mma_commit_pair(&acc_full[slot]);
                    __syncwarp();
                }
            }
            if (lead) mma_commit_pair(&done);
            __syncwarp();
        }
    } else {
        const int quarter = warp & 3, part = (warp - 2) >> 2;  // columns part * 64 .. + 63
        const int t = threadIdx.x - 64;
        const uint32_t lane0 = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t empty0 = map_to(smem_u32(&acc_empty[0]), 0);
        // The scales and biases of a tile, copied while the tile before it is read.
        auto fetch = [&](int tile, int buf) {
            const int m0 = (tile / ctiles) * 256;
            const int c0 = (tile % ctiles) * 256 + static_cast<int>(rank) * 128;
            for (int i = t; i < 3 * 256; i += 32 * kPairReaders) {
                const int m = m0 + (i & 255);
                const bool read = tile < tiles && m < g.M;
                copy4(&scale[buf][i >> 8][i & 255],
                      read ? g.xs + static_cast<int64_t>(x_of(i >> 8)) * g.M + m : g.xs, read);
            }
            for (int i = t; i < 5 * 128; i += 32 * kPairReaders) {
                const int q = i >> 7, c = c0 + (i & 127);
                const float* src = q < 3 ? g.ws + static_cast<int64_t>(w_of(q)) * g.N
                                         : (q == 3 ? g.Sb : g.mb);
                const bool read = tile < tiles && c < g.N && src != nullptr;
                copy4(&chan[buf][q][i & 127], read ? src + c : g.xs, read);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int unit = 0, buf = 0;
        bool alive = true;
        fetch(blockIdx.x / 2, 0);
        for (int tile = blockIdx.x / 2; tile < tiles; tile += pairs, buf ^= 1) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            // every reader's copies are here, and all have left the other buffer
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kPairReaders) : "memory");
            fetch(tile + pairs, buf ^ 1);
            const int m0 = (tile / ctiles) * 256 + part * 64;
            const int n = (tile % ctiles) * 256 + static_cast<int>(rank) * 128 + quarter * 32 + lane;
            const bool in = n < g.N;
            const int lim = g.M - m0;  // columns that are tokens
            const int ch = quarter * 32 + lane;
            float first[64];
#pragma unroll
            for (int p = 0; p < 3; ++p, ++unit) {
                const int slot = unit & 1;
                if (alive)
                    alive = __all_sync(0xffffffffu, mbar_wait(&acc_full[slot], (unit / 2) & 1, ab, 27));
                if (!alive) break;
                tc_fence_after();
                const uint32_t t0 = tmem + lane0 + slot * 256 + part * 64;
                const float4* sc = reinterpret_cast<const float4*>(&scale[buf][p][part * 64]);
                const float b = chan[buf][p][ch], bias = chan[buf][p == 2 ? 4 : 3][ch];
                const float b0 = chan[buf][0][ch];
                float* out = (p == 2 ? g.mz : g.Sz) + static_cast<int64_t>(m0) * g.N + n;
#pragma unroll
                for (int c = 0; c < 64; c += 8) {  // 8 at a time: first[] leaves no room for more
                    uint32_t r[8];
                    tmem_ld8(t0 + c, r);
                    const float4 s0 = sc[c / 4], s1 = sc[c / 4 + 1];
                    const float sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                    tmem_wait_ld();
                    if (p == 0) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            first[c + e] = sv[e] * static_cast<float>(static_cast<int>(r[e]));
                    } else {
                        float z[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            z[e] = fmaf(sv[e] * static_cast<float>(static_cast<int>(r[e])), b,
                                        p == 1 ? fmaf(first[c + e], b0, bias) : bias);
                        if (in && c + 8 <= lim) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                *out = z[e];
                                out += g.N;
                            }
                        } else if (in) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                if (c + e < lim) *out = z[e];
                                out += g.N;
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_read(empty0 + slot * 8);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1 && lane == 0 && !mbar_drain(&done, 0)) atomicCAS(&g_int8_error, 0, 28);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no remote arrival or commit is still due
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---- few tokens or few tiles: a tile's work shared out over a cluster ------------------
constexpr int kSplitThreads = 192;

template <int BN>
struct Split {
    static constexpr int STAGE = 128 * kBK + BN * kBK;
    static constexpr int STAGES = 5;
    static constexpr int COLS = 4 * BN;  // three accumulators; a power of 2
    // the integer sums of the three products, for the exchange, use the stages' room
    static_assert(3 * BN * 128 * 4 <= STAGES * STAGE, "the sums fit");
    static constexpr int SMEM = STAGES * STAGE + 1024;
};

// Work items of CTA `rank` of `ctas`: the list of (product, reduction block) cut evenly.
__device__ __forceinline__ int share(int items, int rank, int ctas) {
    return static_cast<int>(static_cast<int64_t>(items) * rank / ctas);
}

template <int BN>
__global__ void __launch_bounds__(kSplitThreads) int8_split_kernel(const Int8Args g,
                                                                   const __grid_constant__ Maps maps) {
    using P = Split<BN>;
    extern __shared__ char raw[];
    __shared__ __align__(8) uint64_t full[P::STAGES], empty[P::STAGES], done;
    __shared__ uint32_t tmem_base;
    __shared__ int abort_flag;
    __shared__ float scale[3][BN];
    __shared__ int held[8];  // the products that CTA r has sums of, a bit each
    char* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * 128, m0 = blockIdx.y * BN;
    const int ctas = gridDim.z, rank = blockIdx.z;  // the cluster runs along z
    const int kblocks = (g.K + kBK - 1) / kBK;
    const int beg = share(3 * kblocks, rank, ctas), end = share(3 * kblocks, rank + 1, ctas);
    const Abort ab{&abort_flag, 0};

    // item i of this CTA's list into stage s
    auto issue = [&](int i, int s) {
        const int p = i / kblocks, k = (i - p * kblocks) * kBK;
        const uint32_t dst = smem_u32(smem + s * P::STAGE);
        mbar_expect_tx(&full[s], P::STAGE);
        tma_load(dst, &maps.w[w_of(p)], k, n0, &full[s]);
        tma_load(dst + 128 * kBK, &maps.x[x_of(p)], k, m0, &full[s]);
    };
    int issued = beg;  // warp 0, lane 0
    if (threadIdx.x == 0) {
        for (int s = 0; s < P::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        const int give_up = g_int8_force_abort;
        abort_flag = give_up;
        if (give_up) atomicCAS(&g_int8_error, 0, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // this thread's copies use the barriers before any synchronisation of the CTA
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // the first stages fill while the others set up
        wait_for_primary();
        for (; !give_up && issued < end && issued < beg + P::STAGES; ++issued) issue(issued, issued - beg);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_base)),
                     "r"(P::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        launch_dependents();  // behind the allocation: see launch_early
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    wait_for_primary();

    if (warp == 0) {
        // lane 0, which set the barriers up, has filled the first stages already
        int it = __shfl_sync(0xffffffffu, issued, 0) - beg;
        Ring<P::STAGES> ring;
        for (int i = 0; i < it; ++i) ring.next();
#pragma unroll 1
        for (; beg + it < end; ++it, ring.next()) {
            if (!(ring.again ? warp_wait(&empty[ring.s], ring.parity ^ 1u, ab, 11)
                             : __all_sync(0xffffffffu, *ab.flag == 0)))
                break;
            if (lane == 0) issue(beg + it, ring.s);
            __syncwarp();
        }
        // copies still in flight (after an abort) land before the CTA may exit
        for (int i = it > P::STAGES ? it - P::STAGES : 0; i < it; ++i)
            if (!mbar_drain(&full[i % P::STAGES], (i / P::STAGES) & 1) && lane == 0)
                atomicCAS(&g_int8_error, 0, 13);
    } else if (warp == 1) {
        const bool lead = elect_one();
        Ring<P::STAGES> ring;
        int p = beg / kblocks, k = beg - p * kblocks;
        bool first = true;  // of this CTA's blocks of the product
#pragma unroll 1
        for (int i = beg; i < end; ++i, ring.next()) {
            if (!warp_wait(&full[ring.s], ring.parity, ab, 12)) break;
            tc_fence_after();
            const uint32_t idesc = instr_desc(p == 2, 128, BN);
            const uint32_t base = smem_u32(smem + ring.s * P::STAGE);
            const uint64_t a = tile_desc(base), b = tile_desc(base + 128 * kBK);
            const uint32_t d = tmem + p * BN;
            if (lead) {
                mma_i8<false>(d, a, b, idesc, first ? 0u : 1u);
#pragma unroll
                for (int j = 1; j < kBK / 32; ++j) mma_i8<false>(d, a + 2 * j, b + 2 * j, idesc, 1u);
                mma_commit(&empty[ring.s]);
            }
            __syncwarp();
            first = ++k == kblocks;
            if (first) {
                k = 0;
                ++p;
            }
        }
        if (lead) mma_commit(&done);
        __syncwarp();
    } else {
        const int t = threadIdx.x - 64;
        if (t < ctas) {
            const int lo = share(3 * kblocks, t, ctas), hi = share(3 * kblocks, t + 1, ctas);
            int bits = 0;
            for (int p = 0; p < 3; ++p)
                if (lo < hi && hi > p * kblocks && lo < (p + 1) * kblocks) bits |= 1 << p;
            held[t] = bits;
        }
        for (int i = t; i < 3 * BN; i += 128) {
            const int p = i / BN, m = m0 + i % BN;
            scale[p][i % BN] = m < g.M ? g.xs[static_cast<int64_t>(x_of(p)) * g.M + m] : 0.f;
        }
    }
    // accumulators: one thread per channel
    const int quarter = warp & 3;
    const int ch = quarter * 32 + lane, n = n0 + ch;
    const bool reader = warp >= 2;
    float b[3] = {0.f, 0.f, 0.f}, mb = 0.f, Sb = 0.f;
    bool ok = false;
    if (reader) {
        if (n < g.N) {
#pragma unroll
            for (int p = 0; p < 3; ++p) b[p] = g.ws[static_cast<int64_t>(w_of(p)) * g.N + n];
            mb = g.mb ? g.mb[n] : 0.f;
            Sb = g.Sb ? g.Sb[n] : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");  // scale[] and held[] are in place
        ok = __all_sync(0xffffffffu, mbar_wait(&done, 0, ab, 14) && !*ab.flag);
        tc_fence_after();
    }
    const uint32_t t0 = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    auto put = [&](int c, int a0, int a1, int a2) {
        const int m = m0 + c;
        if (n >= g.N || m >= g.M) return;
        const int64_t o = static_cast<int64_t>(m) * g.N + n;
        // rounded as the pair kernel does: a token's result does not depend on the batch
        g.Sz[o] = fmaf(scale[1][c] * static_cast<float>(a1), b[1],
                       fmaf(scale[0][c] * static_cast<float>(a0), b[0], Sb));
        g.mz[o] = fmaf(scale[2][c] * static_cast<float>(a2), b[2], mb);
    };
    if (ctas == 1) {
        if (ok) {
#pragma unroll 1
            for (int c = 0; c < BN && m0 + c < g.M; c += 16) {
                uint32_t r0[16], r1[16], r2[16];
                tmem_ld16(t0 + c, r0);
                tmem_ld16(t0 + BN + c, r1);
                tmem_ld16(t0 + 2 * BN + c, r2);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    put(c + e, static_cast<int>(r0[e]), static_cast<int>(r1[e]),
                        static_cast<int>(r2[e]));
            }
        }
    } else {
        // every copy and MMA of this CTA is complete: its stages hold the sums now
        int* sums = reinterpret_cast<int*>(smem);
        if (reader && ok) {
#pragma unroll 1
            for (int p = 0; p < 3; ++p) {
                if (!(held[rank] >> p & 1)) continue;
#pragma unroll 1
                for (int c = 0; c < BN; c += 16) {
                    uint32_t r[16];
                    tmem_ld16(t0 + p * BN + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sums[(p * BN + c + e) * 128 + ch] = static_cast<int>(r[e]);
                }
            }
        }
        __syncwarp();
        cluster_sync();
        if (reader && ok) {
            // this CTA adds the columns [c0, c1), kWide at a time; the loads of two CTAs
            // are in flight together
            constexpr int kWide = BN / 8;
            const int c0 = share(BN, rank, ctas), c1 = share(BN, rank + 1, ctas);
            const uint32_t at0 = smem_u32(&sums[ch]);
            for (int c = c0; c < c1; c += kWide) {
                int a[3][kWide] = {};
#pragma unroll 1
                for (int r0 = 0; r0 < ctas; r0 += 2) {  // ctas is 2, 4 or 8
                    int v[2][3][kWide];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int bits = held[r0 + r];
                        const uint32_t at = map_to(at0, r0 + r) + c * 512;
#pragma unroll
                        for (int p = 0; p < 3; ++p)
#pragma unroll
                            for (int i = 0; i < kWide; ++i)
                                v[r][p][i] = ld_cluster(at + (p * BN + i) * 512,
                                                        (bits >> p & 1) != 0 && c + i < c1);
                    }
#pragma unroll
                    for (int p = 0; p < 3; ++p)
#pragma unroll
                        for (int i = 0; i < kWide; ++i) a[p][i] += v[0][p][i] + v[1][p][i];
                }
#pragma unroll
                for (int i = 0; i < kWide; ++i)
                    if (c + i < c1) put(c + i, a[0][i], a[1][i], a[2][i]);
            }
        }
        __syncwarp();
        cluster_sync();  // the sums stay until every CTA has read them
    }
    tc_fence_before();
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

// Which kernel, and how a tile of the split kernel is cut. Measured with cold inputs,
// us with about 4 us of the measurement itself:
//   pairs from 96 tiles of 128 x 128 on (32 pairs at work): 1536 x 1024 by K = 512 16
//     against 20 split, 512 x 4096 by 1024 20 against 31; below, fewer pairs win nothing or
//     lose: 512 x 2048 by 2048 27 against 27, 8192 x 128 by 512 18 against 14.
//   BN: 16 while that leaves the reduction four shares or more, else 32, so that the
//     weights are read fewer times: 64 x 4096 by 4096 25 (32 columns, 4 shares) against 31
//     (16, 2 shares); 33 x 1000 by 1000 12 (16 columns) against 14 (32). 64 columns were
//     never faster.
//   shares: up to two CTAs per SM, 3 blocks of the reduction each or more: 1 x 512 by
//     2048 12 with 8, 23 with 1; 16 x 512 by 512 10 with 4, 12 with 1. The exchange of 32
//     columns wants 10 blocks: 128 x 4096 by 4096 33 with 2, 41 with 1; 700 x 700 by 700
//     16 with 2, 14 with 1.
struct Route {
    bool pair;
    int bn, ctas;
};
Route route(int64_t M, int64_t N, int64_t K) {
    const int64_t items = 3 * ((K + kBK - 1) / kBK), ntiles = (N + 127) / 128;
    if (((M + 127) / 128) * ntiles >= 96) return {true, 256, 2};
    Route r{false, ((M + 15) / 16) * ntiles <= kNumSMs / 4 ? 16 : 32, 1};
    const int64_t tiles = ((M + r.bn - 1) / r.bn) * ntiles;
    const int64_t least = r.bn == 16 ? 3 : 10;
    while (r.ctas < 8 && tiles * r.ctas * 2 <= kNumSMs * 2 && items >= r.ctas * 2 * least)
        r.ctas *= 2;
    return r;
}

// The attribute belongs to the current device's copy of the kernel.
template <typename K>
int reserve_smem(K kernel, int bytes, const char* what) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) return TAGI_OK;
    cudaGetLastError();
    set_error("%s: cannot reserve %d bytes of shared memory (%s)", what, bytes,
              cudaGetErrorString(e));
    return TAGI_E_LAUNCH;
}

int launch_pair(const Int8Args& g, const Maps& maps, cudaStream_t st, const char* what) {
    if (const int rc = reserve_smem(int8_pair_kernel, kPairSmem, what)) return rc;
    const int64_t tiles = ((static_cast<int64_t>(g.M) + 255) / 256) * ((g.N + 255) / 256);
    TAGI_REQUIRE(tiles <= INT32_MAX / 2, TAGI_E_UNSUPPORTED, "%s: too many tiles", what);
    const int64_t pairs = tiles < kNumSMs / 2 ? tiles : kNumSMs / 2;
    launch_early(int8_pair_kernel,
                 {dim3(static_cast<unsigned>(2 * pairs)), dim3(kPairThreads), st, kPairSmem,
                  dim3(2)},
                 g, maps);
    count_tc_launch();
    return check_launch(what);
}

template <int BN>
int launch_split(const Int8Args& g, const Maps& maps, int ctas, cudaStream_t st, const char* what) {
    using P = Split<BN>;
    if (const int rc = reserve_smem(int8_split_kernel<BN>, P::SMEM, what)) return rc;
    const int64_t my = (static_cast<int64_t>(g.M) + BN - 1) / BN;
    TAGI_REQUIRE(my <= 65535, TAGI_E_UNSUPPORTED, "%s: too many rows", what);
    launch_early(int8_split_kernel<BN>,
                 {dim3((g.N + 127) / 128, static_cast<unsigned>(my), ctas), dim3(kSplitThreads), st,
                  P::SMEM, dim3(1, 1, ctas)},
                 g, maps);
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
    TAGI_REQUIRE(M >= 0 && N >= 0 && K >= 1 && M <= (1 << 30) && N <= (1 << 30) && K <= 33025,
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
    const Route r = route(M, N, K);
    const int box = r.pair ? 128 : r.bn;
    Maps maps;
    const void* x[3] = {x_m, x_2, x_S};
    const void* w[3] = {w_m, w_2, w_S};
    for (int i = 0; i < 3; ++i)
        TAGI_REQUIRE(encode(&maps.x[i], x[i], M, K, ldx, box) && encode(&maps.w[i], w[i], N, K, ldw, 128),
                     TAGI_E_LAUNCH, "%s: the tensor maps were refused", what);
    const Int8Args g{x_scales, w_scales, mb, Sb, mz, Sz, static_cast<int>(M), static_cast<int>(N),
                     static_cast<int>(K)};
    cudaStream_t st = as_stream(stream);
    if (r.pair) return launch_pair(g, maps, st, what);
    if (r.bn == 16) return launch_split<16>(g, maps, r.ctas, st, what);
    return launch_split<32>(g, maps, r.ctas, st, what);
}
