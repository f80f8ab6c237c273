// Matrix product in e4m3 with a scale for each block of 128, on tcgen05.
//
//   Y[i][j] = sum_b sx[i][b] sw[j / 128][b] sum_{c in block b} xq[i][c] wq[j][c] + bias[j]
//
// A K-block is one scale block: 128 columns = 128 bytes, the SWIZZLE_128B span.
// The tensor core sums within a block (products of e4m3 values are exact in
// fp32), registers across blocks, each block's sum scaled in with one
// multiply-add.  One warp issues TMA loads into a ring of stages, one the MMAs
// of a K-block into the next of several TMEM accumulators, the others drain
// them; the accumulators decouple the two.
//
// Three kernels:
//   * large products (4096 x 8192 x 8192: 250 us, 2.2 PFLOP/s, 290 us where
//     the card is held at its power limit; the tensor core alone takes 169):
//     256 tokens x 256 features on two SMs (cta_group::2),
//     each with half of either operand, which asks 64 bytes a clock of L2 per
//     SM where 128 x 256 on one SM asks 96.  Tokens are the MMA's M (TMEM
//     lanes): a thread holds one token, for which sx sw is one number for all
//     features of a 128-block;
//   * few tokens or few tiles (1 x 151669 x 1536: 40 us, 5.8 TB/s of weights):
//     128 features (lanes) x 16 to 128 tokens
//     (columns) on one SM, K split over a cluster where tiles are few;
//   * 8 tokens and few weights (8 x 4608 x 1536: 4.1 us): registers and
//     mma.sync, one memory round trip.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "drain.h"
#include "fp8.cuh"
#include "per_device.h"
#include "tcgen05.cuh"
#include "xl_device.cuh"
#include "xl_kernels.h"

namespace xl {

namespace {

constexpr int kOpBytes = 128 * kFp8Block;    // 16 KB: 128 rows of an operand's K-block
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 8;                 // portable cluster size
constexpr int kStagePitch = 20;              // floats a row of the store staging: 16 and padding, conflict-free in float4
constexpr int kSmemLimit = 232448;           // 227 KB
constexpr int kBarBytes = 512;

// 256 tokens x 256 features on a pair of SMs.
struct Pair {
    static constexpr int kTokens = 256, kFeatures = 256;  // of the tile; each CTA loads 128 of either
    static constexpr int kStage = 2 * kOpBytes;
    static constexpr int kEpiWarps = 8;                   // each drains 32 lanes x 128 columns
    // the issuing warps are a warpgroup, so that registers can be moved to the epilogue's two
    static constexpr int kEpiFirst = 4;
    static constexpr int kThreads = 32 * (kEpiFirst + kEpiWarps);
    static constexpr int kAccs = 512 / kFeatures;         // TMEM accumulators
    static constexpr int kWarpStore = 32 * kStagePitch + 128;  // floats: a warp's staging rows and its bias
    static constexpr int kStoreBytes = kEpiWarps * kWarpStore * 4;
    // kind::f8f6f4, e4m3 x e4m3, fp32 sums, K-major operands
    static constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(kFeatures >> 3) << 17) |
                                       (static_cast<uint32_t>(kTokens >> 4) << 24);
};

struct LinearParams {
    const float *xs, *ws, *bias;
    void* y;
    int mode, n, m, blocks;     // blocks: K-blocks
    int stages;
    int split;                  // CTAs of a cluster that share a tile's K-blocks (features on lanes)
    int tiles_n, tiles_m;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    return a;
}
// Every thread of every CTA of a cluster comes here on every path, so it ends.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A whole warp waits, and agrees on whether the wait ended in time.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity) || wait_bar(bar, parity, nullptr));
}

template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
            "{%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_e4m3(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Arrives on `bar` (in both CTAs of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if (CG == 1)
        mma_commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"(static_cast<uint16_t>(3))
            : "memory");
}

// 32 columns of the warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// The loads so far have landed; naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait64(uint32_t (&a)[32], uint32_t (&b)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                   "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]),
                   "+r"(a[15]), "+r"(a[16]), "+r"(a[17]), "+r"(a[18]), "+r"(a[19]), "+r"(a[20]), "+r"(a[21]),
                   "+r"(a[22]), "+r"(a[23]), "+r"(a[24]), "+r"(a[25]), "+r"(a[26]), "+r"(a[27]), "+r"(a[28]),
                   "+r"(a[29]), "+r"(a[30]), "+r"(a[31]), "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]),
                   "+r"(b[5]), "+r"(b[6]), "+r"(b[7]), "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]), "+r"(b[12]),
                   "+r"(b[13]), "+r"(b[14]), "+r"(b[15]), "+r"(b[16]), "+r"(b[17]), "+r"(b[18]), "+r"(b[19]),
                   "+r"(b[20]), "+r"(b[21]), "+r"(b[22]), "+r"(b[23]), "+r"(b[24]), "+r"(b[25]), "+r"(b[26]),
                   "+r"(b[27]), "+r"(b[28]), "+r"(b[29]), "+r"(b[30]), "+r"(b[31])
                 :
                 : "memory");
}
__device__ __forceinline__ unsigned long long pack2(uint32_t lo, uint32_t hi) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ float2 unpack2(unsigned long long d) {
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(d));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}
__device__ __forceinline__ void fma2(unsigned long long& acc, unsigned long long a, unsigned long long b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

// acc[first ..] += s * 32 columns
__device__ __forceinline__ void scale_in(unsigned long long (&acc)[64], int first, const uint32_t (&r)[32],
                                         unsigned long long s2) {
#pragma unroll
    for (int i = 0; i < 16; ++i) fma2(acc[first + i], pack2(r[2 * i], r[2 * i + 1]), s2);
}

// v / (1 + e^-v) = v e^v / (1 + e^v), within 7 ulp.  With e^-|v| as the square of h = e^(-|v| / 2) no step leaves the
// floats' range before the result does (e^-v passes it at v = -89, where v e^v has not, and the fast division gives 0 for
// divisors above 2^126); without a branch, of which a tile's store would hold one an output (13.6 us of a 512 x 8192 x 1536
// product became 16.9).
__device__ __forceinline__ float silu_fast(float v) {
    const float h = expf(-0.5f * fabsf(v)), e = h * h;
    return __fdividef(v < 0.0f ? v * h * h : v, 1.0f + e);
}

template <typename T>
__device__ __forceinline__ void put(T* dst, float v, int mode) {
    *dst = from_float<T>(mode == kGemvResidual ? to_float(*dst) + v : v);
}

// 32 tokens x 128 features in registers (a token a lane) to y, 16 outputs a
// row at a time through the warp's staging rows, so that stores are 16 bytes
// a lane along the rows.  bias: the warp's 128 values in shared memory.
template <typename T, int MODE>
__device__ __forceinline__ void store_rows(const unsigned long long (&acc)[64], const LinearParams& p, int tok0, int j0,
                                           float* st, const float4* bias, int lane) {
    constexpr bool swiglu = MODE == kGemvSwiGLU;
    const int wide = swiglu ? p.m / 2 : p.m;
    const bool vec = (static_cast<size_t>(wide) * sizeof(T)) % 16 == 0;
    const int rows = min(32, p.n - tok0);
    T* y = static_cast<T*>(p.y);
    constexpr int kPer = 16 / sizeof(T);  // outputs of a 16-byte store
    float4* row = reinterpret_cast<float4*>(st + lane * kStagePitch);
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
        if (swiglu && ch >= 4) break;
        const int o0 = (swiglu ? j0 / 2 : j0) + ch * 16;
        if (o0 >= wide) break;
        if (swiglu) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 b = bias[(ch & 3) * 8 + 2 * i + h];
                    const float2 e = unpack2(acc[(ch & 3) * 16 + 4 * i + 2 * h]), f = unpack2(acc[(ch & 3) * 16 + 4 * i + 2 * h + 1]);
                    v[2 * h] = silu_fast(e.x + b.x) * (e.y + b.y);
                    v[2 * h + 1] = silu_fast(f.x + b.z) * (f.y + b.w);
                }
                row[i] = make_float4(v[0], v[1], v[2], v[3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 b = bias[ch * 4 + i];
                const float2 e = unpack2(acc[ch * 8 + 2 * i]), f = unpack2(acc[ch * 8 + 2 * i + 1]);
                row[i] = make_float4(e.x + b.x, e.y + b.y, f.x + b.z, f.y + b.w);
            }
        }
        __syncwarp();
        // what y holds is read for all rows before the first is written: one memory round trip, not one a row
        if (vec && o0 + 16 <= wide) {
            constexpr int kLanes = 16 / kPer, kTurns = kLanes;  // lanes a row; rows 32 / kLanes at a time
            T* dst = y + static_cast<size_t>(tok0 + lane / kLanes) * wide + o0 + lane % kLanes * kPer;
            const size_t turn = static_cast<size_t>(32 / kLanes) * wide;
            if constexpr (MODE == kGemvResidual) {
                uint4 old[kTurns];
#pragma unroll
                for (int i = 0; i < kTurns; ++i) {
                    old[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (i * (32 / kLanes) + lane / kLanes < rows) old[i] = *reinterpret_cast<const uint4*>(dst + i * turn);
                }
#pragma unroll
                for (int i = 0; i < kTurns; ++i) {
                    const int r = i * (32 / kLanes) + lane / kLanes;
                    if (r < rows) {
                        const float* src = st + r * kStagePitch + lane % kLanes * kPer;
                        T* e = reinterpret_cast<T*>(&old[i]);
#pragma unroll
                        for (int k = 0; k < kPer; ++k) e[k] = from_float<T>(to_float(e[k]) + src[k]);
                        *reinterpret_cast<uint4*>(dst + i * turn) = old[i];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kTurns; ++i) {
                    const int r = i * (32 / kLanes) + lane / kLanes;
                    if (r < rows) {
                        const float* src = st + r * kStagePitch + lane % kLanes * kPer;
                        uint4 out;
                        T* e = reinterpret_cast<T*>(&out);
#pragma unroll
                        for (int k = 0; k < kPer; ++k) e[k] = from_float<T>(src[k]);
                        *reinterpret_cast<uint4*>(dst + i * turn) = out;
                    }
                }
            }
        } else {
            // 16 lanes a row, or rows of whole words: 8 lanes with 2 outputs (16-bit y)
            const bool two = sizeof(T) == 2 && wide % 2 == 0;
            const int per = two ? 2 : 1, lanes = 16 / per, apart = 32 / lanes;
            const int r0 = lane / lanes, c = lane % lanes * per;
            T* dst = y + static_cast<size_t>(tok0 + r0) * wide + o0 + c;
            const float* src = st + r0 * kStagePitch + c;
            const size_t turn = static_cast<size_t>(apart) * wide;
            const int mine = o0 + c < wide ? (rows - r0 + apart - 1) / apart : 0;
            if (MODE == kGemvResidual) {
#pragma unroll 1
                for (int t0 = 0; t0 < mine; t0 += 8) {
                    float old[8];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (half >= per) break;
#pragma unroll
                        for (int i = 0; i < 8; ++i) old[i] = t0 + i < mine ? to_float(dst[(t0 + i) * turn + half]) : 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (t0 + i < mine)
                                dst[(t0 + i) * turn + half] = from_float<T>(old[i] + src[(t0 + i) * apart * kStagePitch + half]);
                    }
                }
            } else if (two) {
                if constexpr (sizeof(T) == 2) {
#pragma unroll 4
                    for (int i = 0; i < mine; ++i) {
                        const float* v = src + i * apart * kStagePitch;
                        *reinterpret_cast<uint32_t*>(dst + i * turn) = pack_pair(v[0], v[1], T{});
                    }
                }
            } else {
#pragma unroll 4
                for (int i = 0; i < mine; ++i) dst[i * turn] = from_float<T>(src[i * apart * kStagePitch]);
            }
        }
        __syncwarp();
    }
}

// MODE at compile time: a tile's store runs once or a few times a call, and the code of the other modes beside it cost
// instruction fetch.
template <typename T, int MODE>
__global__ void __launch_bounds__(Pair::kThreads, 1)
    linear_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                           const LinearParams p) {
    extern __shared__ __align__(1024) char smem_raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* store = reinterpret_cast<float*>(ring + p.stages * Pair::kStage);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(store) + Pair::kStoreBytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* done = empty + kMaxStages;   // an accumulator holds a K-block's sums
    uint64_t* freed = done + Pair::kAccs;  // its columns have been read, in both CTAs (see DrainTurn for their number)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(freed + 2 * Pair::kAccs);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());
    const int unit = static_cast<int>(blockIdx.x) / 2, units = static_cast<int>(gridDim.x) / 2;
    const int tiles = p.tiles_n * p.tiles_m;

    if (warp == 0) {
        if (elect_one()) asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&map_x), "l"(&map_w) : "memory");
        if (lane < p.stages) {
            mbar_init(&full[lane], 1);
            mbar_init(&empty[lane], 1);
        }
        if (lane < Pair::kAccs) mbar_init(&done[lane], 1);
        if (lane < 2 * Pair::kAccs) mbar_init(&freed[lane], 2 * Pair::kEpiWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();  // the peer's barriers are set up before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    // The epilogue needs 128 sums and 64 columns in flight a thread: 384 threads launch with 168 registers, the
    // issuing warpgroup keeps 40, the others take 232 (128 x 40 + 256 x 232 = 384 x 168).
    if (warp < Pair::kEpiFirst) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // Token tiles advance fastest: the CTAs that run together share W tiles and, over the whole product, either
    // operand stays in L2.  Both issuing warps run their loops converged and elect one lane to issue.
    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0, issued = 0;
        bool ok = true;
        const uint32_t bar0 = cluster_addr(smem_u32(full), 0);  // both CTAs' copies are counted in the first one
        for (int t = unit; t < tiles && ok; t += units) {
            const int y_x = t % p.tiles_n * Pair::kTokens + rank * 128, y_w = t / p.tiles_n * Pair::kFeatures + rank * 128;
            for (int kb = 0; kb < p.blocks; ++kb) {
                if (!wait_warp(&empty[s], ph ^ 1u)) {
                    ok = false;
                    break;
                }
                const uint32_t st = smem_u32(ring + s * Pair::kStage);
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * Pair::kStage);
                    load_tile<2>(st, &map_x, kb * kFp8Block, y_x, bar0 + 8 * s);
                    load_tile<2>(st + kOpBytes, &map_w, kb * kFp8Block, y_w, bar0 + 8 * s);
                }
                __syncwarp();
                ++issued;
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
        }
        if (!ok && rank == 0) {
            // the copies in flight land before the CTAs leave
            for (uint32_t i = 0; i < min(issued, static_cast<uint32_t>(p.stages)); ++i) {
                if (s == 0) s = p.stages, ph ^= 1u;
                --s;
                wait_warp(&full[s], ph);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            int s = 0, a = 0;
            uint32_t ph = 0, pa = 0;
            bool ok = true, any = false;
            for (int t = unit; t < tiles && ok; t += units) {
                for (int kb = 0; kb < p.blocks; ++kb) {
                    if (!wait_warp(&full[s], ph) || !wait_warp(&freed[a], pa ^ 1u)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t st = smem_u32(ring + s * Pair::kStage);
                    const uint64_t dx = umma_desc(st), dw = umma_desc(st + kOpBytes);
                    const uint32_t acc = tmem + static_cast<uint32_t>(a * Pair::kFeatures);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)  // 32 columns = 32 bytes each
                            mma_e4m3<2>(acc, dx + 2 * ks, dw + 2 * ks, Pair::kIdesc, ks != 0);
                        commit<2>(&done[a]);
                        commit<2>(&empty[s]);
                    }
                    __syncwarp();
                    any = true;
                    if (++s == p.stages) s = 0, ph ^= 1u;
                    if (++a == Pair::kAccs) a = 0, pa ^= 1u;
                }
            }
            if (!ok && any) {  // the MMAs in flight end before the TMEM is given back
                if (a == 0) a = Pair::kAccs, pa ^= 1u;
                wait_warp(&done[a - 1], pa);
            }
        }
    } else if (warp >= Pair::kEpiFirst) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // TMEM lanes are a warp's by its number modulo 4
        const int q = warp & 3, half = (warp - Pair::kEpiFirst) >> 2;
        float* st = store + (warp - Pair::kEpiFirst) * Pair::kWarpStore;
        float* sb = st + 32 * kStagePitch;
        DrainTurn<Pair::kAccs> turn;
        const uint32_t freed0 = cluster_addr(smem_u32(freed), 0);
        for (int t = unit; t < tiles; t += units) {
            const int tok0 = t % p.tiles_n * Pair::kTokens + rank * 128 + 32 * q;
            const int j0 = t / p.tiles_n * Pair::kFeatures + 128 * half;
            const bool work = tok0 < p.n && j0 < p.m;  // else the warp only keeps the accumulators moving
            const float* xs = p.xs + static_cast<size_t>(min(tok0 + lane, p.n - 1)) * p.blocks;
            const float* ws = p.ws + static_cast<size_t>(min(j0, p.m - 1) / kFp8Block) * p.blocks;
            float bias[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = j0 + 32 * i + lane;
                bias[i] = p.bias && j < p.m ? p.bias[j] : 0.0f;
            }
            unsigned long long acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            float sx = xs[0], sw = ws[0];
            bool ready = mbar_test_wait(&done[turn.acc], turn.parity);
#pragma unroll 1
            for (int kb = 0; kb < p.blocks; ++kb) {
                const float s = sx * sw;
                const int next = min(kb + 1, p.blocks - 1);
                sx = xs[next], sw = ws[next];
                if (turn.ok && !__all_sync(0xffffffffu, ready))
                    turn.waited(wait_warp(&done[turn.acc], turn.parity));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const bool drain = work && turn.ok;
                const unsigned long long s2 = pack2(__float_as_uint(s), __float_as_uint(s));
                uint32_t r0[32], r1[32];
                if (drain) {
                    const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) +
                                        static_cast<uint32_t>(turn.acc * Pair::kFeatures + 128 * half);
                    // two rounds of 64 columns in flight; the accumulator is handed back before the last sums
                    tmem_load32(ta, r0);
                    tmem_load32(ta + 32, r1);
                    tmem_wait64(r0, r1);
                    scale_in(acc, 0, r0, s2);
                    tmem_load32(ta + 64, r0);
                    scale_in(acc, 16, r1, s2);
                    tmem_load32(ta + 96, r1);
                    tmem_wait64(r0, r1);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (elect_one())
                    // only TMEM reads are ordered by this arrival (the fence above); a cluster-wide release of
                    // memory would cost over 1000 clocks a K-block
                    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(freed0 + 8 * turn.acc) : "memory");
                turn.next();
                if (kb + 1 < p.blocks) ready = mbar_test_wait(&done[turn.acc], turn.parity);  // asked early: the answer comes behind the sums
                if (drain) {
                    scale_in(acc, 32, r0, s2);
                    scale_in(acc, 48, r1, s2);
                }
            }
            if (!turn.ok) {  // a wait ran out: the results say so
#pragma unroll
                for (int i = 0; i < 64; ++i) acc[i] = 0x7fffffff7fffffffull;
            }
            if (work) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sb[32 * i + lane] = bias[i];
                __syncwarp();
                store_rows<T, MODE>(acc, p, tok0, j0, st, reinterpret_cast<const float4*>(sb), lane);
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    __syncwarp();
    __syncthreads();
    cluster_sync();  // no CTA leaves while the other may reach its shared memory
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

using LinearKernel = void (*)(CUtensorMap, CUtensorMap, LinearParams);

// `allowed`: the devices on which the kernel may already have this much shared memory.
cudaError_t launch_linear(LinearKernel kernel, std::atomic<unsigned long long>& allowed, const CUtensorMap& mx,
                          const CUtensorMap& mw, const LinearParams& p, int grid, int threads, int cluster, int smem,
                          cudaStream_t s) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kernel, mx, mw, p);
}

template <typename T, int MODE>
cudaError_t launch_pairs(const CUtensorMap& mx, const CUtensorMap& mw, const LinearParams& p, int grid, cudaStream_t s) {
    // the warpgroups' register shares have to fit what the CTA launches with, or the larger one never comes
    static const bool fits = [] {
        cudaFuncAttributes a{};
        return cudaFuncGetAttributes(&a, linear_fp8_pair_kernel<T, MODE>) == cudaSuccess &&
               a.numRegs * Pair::kThreads >= 128 * 40 + 256 * 232;
    }();
    if (!fits) return cudaErrorInvalidConfiguration;
    static std::atomic<unsigned long long> allowed{0};
    return launch_linear(linear_fp8_pair_kernel<T, MODE>, allowed, mx, mw, p, grid, Pair::kThreads, 2,
                         p.stages * Pair::kStage + Pair::kStoreBytes + kBarBytes + 1024, s);
}

// ---- few tokens or tiles: features on the TMEM lanes ----
//
// The operands change places: 128 features are the MMA's M, the tokens its N
// (16 to 128).  A K-block then leaves few columns to drain, a lane's
// results of one token lie next to its neighbours' in y, and the tensor core
// takes a K-block in the time its weights take to arrive.  Fewer tiles than
// SMs split K over the CTAs of a cluster, whose partial tiles meet in
// distributed shared memory.

template <int N>
struct Few {
    static constexpr int kAccs = N >= 64 ? 4 : 8;
    static constexpr int kColumns = kAccs * N;
    static constexpr int kRound = N < 64 ? N : 64;     // columns drained at a time
    static constexpr int kCtas = N == 128 ? 1 : 2;     // an SM holds at least, by registers
    static constexpr int kThreads = 192;
    static constexpr int kStage = kOpBytes + N * kFp8Block;
    static constexpr int kScaleBytes = 4 * N * 4;  // a warp's N scales
    static constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
};

// N TMEM columns of the warp's 32 lanes, 16 at a time.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

template <int N, typename T>
__global__ void __launch_bounds__(Few<N>::kThreads, Few<N>::kCtas)
    linear_fp8_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                          const LinearParams p) {
    using F = Few<N>;
    extern __shared__ __align__(1024) char smem_raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* scales = reinterpret_cast<float*>(ring + p.stages * F::kStage);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(scales) + F::kScaleBytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* done = empty + kMaxStages;
    uint64_t* freed = done + F::kAccs;
    uint64_t* quiet = freed + 2 * F::kAccs;  // both issuing warps have stopped
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(quiet + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = p.split > 1 ? cluster_rank() : 0u;
    const int unit = static_cast<int>(blockIdx.x) / p.split, units = static_cast<int>(gridDim.x) / p.split;
    const int tiles = p.tiles_n * p.tiles_m;
    const int kb0 = static_cast<int>(static_cast<long long>(rank) * p.blocks / p.split);
    const int kb1 = static_cast<int>(static_cast<long long>(rank + 1) * p.blocks / p.split);

    if (warp == 0) {
        if (elect_one()) asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&map_x), "l"(&map_w) : "memory");
        if (lane < p.stages) {
            mbar_init(&full[lane], 1);
            mbar_init(&empty[lane], 1);
        }
        if (lane < F::kAccs) mbar_init(&done[lane], 1);
        if (lane < 2 * F::kAccs) mbar_init(&freed[lane], 4);
        if (lane == 0) mbar_init(quiet, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "n"(F::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 0, issued = 0;
        bool ok = true;
        for (int t = unit; t < tiles && ok; t += units) {
            const int tn = t % p.tiles_n, tm = t / p.tiles_n;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_warp(&empty[s], ph ^ 1u)) {
                    ok = false;
                    break;
                }
                const uint32_t st = smem_u32(ring + s * F::kStage);
                if (elect_one()) {
                    mbar_expect_tx(&full[s], F::kStage);
                    load_tile<1>(st, &map_w, kb * kFp8Block, tm * 128, smem_u32(&full[s]));
                    load_tile<1>(st + kOpBytes, &map_x, kb * kFp8Block, tn * N, smem_u32(&full[s]));
                }
                __syncwarp();
                ++issued;
                if (++s == p.stages) s = 0, ph ^= 1u;
            }
        }
        if (!ok) {
            // the copies in flight land before the CTA leaves
            for (uint32_t i = 0; i < min(issued, static_cast<uint32_t>(p.stages)); ++i) {
                if (s == 0) s = p.stages, ph ^= 1u;
                --s;
                wait_warp(&full[s], ph);
            }
        }
        __syncwarp();
        if (elect_one()) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(quiet)) : "memory");
    } else if (warp == 1) {
        int s = 0, a = 0;
        uint32_t ph = 0, pa = 0;
        bool ok = true, any = false;
        for (int t = unit; t < tiles && ok; t += units) {
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_warp(&freed[a], pa ^ 1u) || !wait_warp(&full[s], ph)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t st = smem_u32(ring + s * F::kStage);
                const uint64_t dw = umma_desc(st), dx = umma_desc(st + kOpBytes);
                const uint32_t acc = tmem + static_cast<uint32_t>(a * N);
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) mma_e4m3<1>(acc, dw + 2 * ks, dx + 2 * ks, F::kIdesc, ks != 0);
                    commit<1>(&empty[s]);
                    commit<1>(&done[a]);
                }
                __syncwarp();
                any = true;
                if (++s == p.stages) s = 0, ph ^= 1u;
                if (++a == F::kAccs) a = 0, pa ^= 1u;
            }
        }
        if (!ok && any) {  // the MMAs in flight end before the TMEM is given back
            if (a == 0) a = F::kAccs, pa ^= 1u;
            wait_warp(&done[a - 1], pa);
        }
        __syncwarp();
        if (elect_one()) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(quiet)) : "memory");
    } else {
        const int q = warp & 3;
        float* sc = scales + (warp - 2) * N;
        DrainTurn<F::kAccs> turn;
        constexpr int kLots = (N + 31) / 32;
        for (int t = unit; t < tiles; t += units) {
            const int tok0 = t % p.tiles_n * N, tm = t / p.tiles_n, rows = min(N, p.n - tok0);
            const float* xs[kLots];
#pragma unroll
            for (int i = 0; i < kLots; ++i) xs[i] = p.xs + static_cast<size_t>(min(tok0 + 32 * i + lane, p.n - 1)) * p.blocks;
            const float* ws = p.ws + static_cast<size_t>(tm) * p.blocks;
            const int j = tm * 128 + 32 * q + lane;
            const float bias = p.bias && j < p.m ? p.bias[j] : 0.0f;
            unsigned long long acc[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) acc[i] = 0;
            float sx[kLots], sw = ws[kb0];
#pragma unroll
            for (int i = 0; i < kLots; ++i) sx[i] = xs[i][kb0];
            bool ready = mbar_test_wait(&done[turn.acc], turn.parity);
#pragma unroll 1
            for (int kb = kb0; kb < kb1; ++kb) {
#pragma unroll
                for (int i = 0; i < kLots; ++i)
                    if (32 * i + lane < N) sc[32 * i + lane] = sx[i] * sw;
                const int next = min(kb + 1, kb1 - 1);
                sw = ws[next];
#pragma unroll
                for (int i = 0; i < kLots; ++i) sx[i] = xs[i][next];
                __syncwarp();
                if (turn.ok && !__all_sync(0xffffffffu, ready))
                    turn.waited(wait_warp(&done[turn.acc], turn.parity));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t r[F::kRound];
                const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) + static_cast<uint32_t>(turn.acc * N);
#pragma unroll
                for (int c = 0; c < N; c += F::kRound) {
                    if (turn.ok) {
#pragma unroll
                        for (int i = 0; i < F::kRound; i += 16) tmem_load16(ta + c + i, r + i);
#pragma unroll
                        for (int i = 0; i < F::kRound; i += 16) tmem_wait16(r + i);
                    }
                    if (c + F::kRound == N) {  // handed back before the last sums
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (elect_one())
                            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&freed[turn.acc])) : "memory");
                        turn.next();
                        if (kb + 1 < kb1) ready = mbar_test_wait(&done[turn.acc], turn.parity);
                    }
                    if (turn.ok) {
#pragma unroll
                        for (int i = 0; i < F::kRound / 4; ++i) {
                            const ulonglong2 s4 = reinterpret_cast<const ulonglong2*>(sc)[c / 4 + i];
                            fma2(acc[c / 2 + 2 * i], pack2(r[4 * i], r[4 * i + 1]), s4.x);
                            fma2(acc[c / 2 + 2 * i + 1], pack2(r[4 * i + 2], r[4 * i + 3]), s4.y);
                        }
                    }
                }
                __syncwarp();
            }
            if (!turn.ok) {  // a wait ran out: the results say so
#pragma unroll
                for (int i = 0; i < N / 2; ++i) acc[i] = 0x7fffffff7fffffffull;
            }
            if (p.split == 1) {
                T* y = static_cast<T*>(p.y);
                const bool swiglu = p.mode == kGemvSwiGLU;
#pragma unroll
                for (int i0 = 0; i0 < N; i0 += 16) {
                    // what y holds is read for 16 tokens before the first is written
                    float old[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        old[i] = 0.0f;
                        if (p.mode == kGemvResidual && i0 + i < rows && j < p.m)
                            old[i] = to_float(y[static_cast<size_t>(tok0 + i0 + i) * p.m + j]);
                    }
#pragma unroll
                    for (int i = i0; i < i0 + 16; ++i) {
                        const size_t row = static_cast<size_t>(tok0 + i);
                        const float2 v2 = unpack2(acc[i / 2]);
                        const float v = (i & 1 ? v2.y : v2.x) + bias;
                        if (i >= rows) {
                        } else if (swiglu) {
                            const float c = __shfl_xor_sync(0xffffffffu, v, 1);
                            if (!(lane & 1) && j < p.m) y[row * (p.m >> 1) + (j >> 1)] = from_float<T>(silu_fast(v) * c);
                        } else if (j < p.m) {
                            y[row * p.m + j] = from_float<T>(old[i - i0] + v);
                        }
                    }
                }
            } else {
                // every K-block of this CTA has been multiplied: the ring is free for the partial tile [tokens][128]; where a
                // wait ran out, only once the issuing warps have stopped and their copies have landed
                for (int i = 0; i < 8 && !turn.ok; ++i)
                    if (wait_warp(quiet, 0)) break;
                float* part = reinterpret_cast<float*>(ring);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float2 v2 = unpack2(acc[i / 2]);
                    if (i < rows) part[i * 128 + 32 * q + lane] = i & 1 ? v2.y : v2.x;
                }
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (p.split > 1) {
        __syncwarp();
        cluster_sync();
        // A cluster has one tile; this CTA finishes its share of the (token, 4 features) pieces.
        const uint32_t part = smem_u32(ring);
        const int tok0 = unit % p.tiles_n * N, tm = unit / p.tiles_n;
        const int pieces = min(N, p.n - tok0) * 32, e1 = static_cast<int>(static_cast<long long>(rank + 1) * pieces / p.split);
        T* y = static_cast<T*>(p.y);
        for (int e = static_cast<int>(static_cast<long long>(rank) * pieces / p.split) + threadIdx.x; e < e1; e += F::kThreads) {
            const int tok = tok0 + (e >> 5), j = tm * 128 + (e & 31) * 4;
            float4 v[kMaxSplit];
#pragma unroll
            for (int k = 0; k < kMaxSplit; ++k) {
                v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (k < p.split)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w)
                                 : "r"(cluster_addr(part + static_cast<uint32_t>(e) * 16, k))
                                 : "memory");
            }
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = p.bias && j + i < p.m ? p.bias[j + i] : 0.0f;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kMaxSplit; ++k) sum[0] += v[k].x, sum[1] += v[k].y, sum[2] += v[k].z, sum[3] += v[k].w;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += sum[i];
            if (p.mode == kGemvSwiGLU) {
                T* dst = y + static_cast<size_t>(tok) * (p.m >> 1) + (j >> 1);
                if (j < p.m) dst[0] = from_float<T>(silu_fast(o[0]) * o[1]);
                if (j + 2 < p.m) dst[1] = from_float<T>(silu_fast(o[2]) * o[3]);
            } else {
                T* dst = y + static_cast<size_t>(tok) * p.m + j;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p.mode == kGemvResidual && j + i < p.m) o[i] += to_float(dst[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (j + i < p.m) dst[i] = from_float<T>(o[i]);
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (p.split > 1) cluster_sync();  // no CTA leaves while another may read its shared memory
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(F::kColumns) : "memory");
    }
}

// ---- few tokens and weights: the weights stream through registers ----

// 16 bytes of a row from column c on, zeros past k (the bytes between k and the row's pitch are not touched).
__device__ __forceinline__ uint4 load_row16(const uint8_t* row, int c, int k) {
    if (c + 16 <= k) return *reinterpret_cast<const uint4*>(row + c);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    for (int i = 0; i < 16; ++i)
        if (c + i < k) w[i >> 2] |= static_cast<uint32_t>(row[c + i]) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void mma_16x8x32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One K-block's operands of a lane: weight rows g and g + 8 and the token's
// row, 2 x 16 bytes each.  A lane reads 16 consecutive bytes where the MMA's
// layout wants 4 x 4: the columns are permuted alike in both operands, so the
// sums are the same.
struct StreamBlock {
    uint4 a[2][2], b[2];
    float s[2];
};

struct StreamParams {
    const uint8_t *xq, *wq;
    size_t ldx, ldw;
    const float *xs, *ws, *bias;
    void* y;
    int mode, n, m, k, blocks;
};

constexpr int kStreamTokens = 8;            // columns of the MMA
constexpr long long kStreamBytes = 9 << 20;  // most weights: beyond, TMA and tcgen05 take less (see launch_tokens)
constexpr int kStreamDepth = 4;             // K-blocks of a warp in flight
constexpr int kStreamWarps = 16;            // most

// 16 weight rows a CTA, its warps share the K-blocks and add up through shared
// memory.  No TMEM, no barriers but one: the product of a small decode step is
// one memory round trip, and every load of a CTA is in flight at once.
template <typename T>
__global__ void __launch_bounds__(32 * kStreamWarps) linear_fp8_stream_kernel(const StreamParams p) {
    constexpr int kPitch = kStreamTokens + 1;
    __shared__ float part[kStreamWarps * 16 * kPitch];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = static_cast<int>(blockDim.x >> 5);
    const int g = lane >> 2, t = lane & 3, row0 = static_cast<int>(blockIdx.x) * 16;
    const uint8_t* wr[2];
    const float* sx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        wr[i] = p.wq + static_cast<size_t>(min(row0 + g + 8 * i, p.m - 1)) * p.ldw;
        sx[i] = p.xs + static_cast<size_t>(min(2 * t + i, p.n - 1)) * p.blocks;
    }
    const uint8_t* xr = p.xq + static_cast<size_t>(min(g, p.n - 1)) * p.ldx;
    const float* sw = p.ws + static_cast<size_t>(row0 / kFp8Block) * p.blocks;
    auto load = [&](StreamBlock& o, int kb) {
        if (kb >= p.blocks) return;
        const int c = kb * kFp8Block + 16 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) o.a[i][h] = load_row16(wr[i], c + 64 * h, p.k);
            o.b[h] = load_row16(xr, c + 64 * h, p.k);
        }
        const float w = sw[kb];
#pragma unroll
        for (int j = 0; j < 2; ++j) o.s[j] = sx[j][kb] * w;
    };
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    StreamBlock ring[kStreamDepth];
#pragma unroll
    for (int d = 0; d < kStreamDepth; ++d) load(ring[d], warp + d * warps);
    for (int kb = warp; kb < p.blocks; kb += kStreamDepth * warps) {
#pragma unroll
        for (int d = 0; d < kStreamDepth; ++d) {
            const int at = kb + d * warps;
            if (at < p.blocks) {
                const StreamBlock& o = ring[d];
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma_16x8x32(c, o.a[0][h].x, o.a[1][h].x, o.a[0][h].y, o.a[1][h].y, o.b[h].x, o.b[h].y);
                    mma_16x8x32(c, o.a[0][h].z, o.a[1][h].z, o.a[0][h].w, o.a[1][h].w, o.b[h].z, o.b[h].w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = fmaf(c[j], o.s[j & 1], acc[j]);
                load(ring[d], at + kStreamDepth * warps);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[(warp * 16 + g + (j >> 1) * 8) * kPitch + 2 * t + (j & 1)] = acc[j];
    __syncthreads();
    const int step = p.mode == kGemvSwiGLU ? 2 : 1, outs = 16 / step, wide = p.m / step;
    T* y = static_cast<T*>(p.y);
    for (int e = threadIdx.x; e < outs * p.n; e += blockDim.x) {
        const int tok = e / outs, r = (e - tok * outs) * step, j = row0 + r;
        if (j >= p.m) continue;
        float v[2] = {0.0f, 0.0f};
        for (int i = 0; i < step; ++i) {
            for (int w = 0; w < warps; ++w) v[i] += part[(w * 16 + r + i) * kPitch + tok];
            if (p.bias) v[i] += p.bias[j + i];
        }
        put(y + static_cast<size_t>(tok) * wide + j / step, step == 2 ? silu_fast(v[0]) * v[1] : v[0], p.mode);
    }
}

template <typename T>
cudaError_t launch_stream(const StreamParams& p, int num_sms, cudaStream_t s) {
    // enough warps to cover a memory round trip with the CTAs an SM holds; more where the rows are few
    int warps = 4;
    while (warps < kStreamWarps && 2 * warps <= p.blocks && static_cast<long long>(p.m / 16) * warps < 16ll * num_sms)
        warps *= 2;
    count_launch();
    linear_fp8_stream_kernel<T><<<(p.m - 1) / 16 + 1, 32 * warps, 0, s>>>(p);
    return cudaGetLastError();
}


int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Clusters of `split` CTAs that the current device runs at once with a CTA an SM.
template <typename Kernel>
int clusters_at_once(Kernel kernel, int split, int threads) {
    int n = 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(split));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = kSmemLimit;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// K split over how many CTAs: as many as run at once, powers of two.
template <int N, typename T>
int few_split(long long tiles, int blocks, int num_sms) {
    static PerDevice at_once[3];  // clusters of 2, 4, 8
    auto clusters = [&](int i, int s) {
        int dev = -1;
        if (cudaGetDevice(&dev) != cudaSuccess) return 0;
        return at_once[i].get(dev, [&] { return clusters_at_once(linear_fp8_few_kernel<N, T>, s, Few<N>::kThreads); });
    };
    int split = 1;
    for (int i = 0, s = 2; s <= kMaxSplit && s <= blocks; ++i, s *= 2) {
        // two CTAs an SM (fewer stages, see below) leave room to place the clusters of one wave of CTAs
        const bool fits = Few<N>::kCtas > 1 ? tiles * s <= num_sms
                                            : tiles <= clusters(i, s);
        if (!fits) break;
        split = s;
    }
    return split;
}

template <int N, typename T>
cudaError_t launch_features_on_lanes(LinearParams& p, const uint8_t* xq, size_t ldx, const uint8_t* wq, size_t ldw, int k,
                                     int num_sms, cudaStream_t s) {
    using F = Few<N>;
    p.tiles_n = cdiv(p.n, N);
    p.tiles_m = cdiv(p.m, 128);
    const long long tiles = static_cast<long long>(p.tiles_n) * p.tiles_m;
    p.stages = std::min(kMaxStages, (kSmemLimit - 1024 - kBarBytes - F::kScaleBytes) / F::kStage);
    p.split = few_split<N, T>(tiles, p.blocks, num_sms);
    // A CTA of a split tile has few K-blocks and takes no more stages than those: several share an SM, so that the
    // clusters run at once (36 clusters of 4 with an SM a CTA did not: 8.2 us where one wave takes 5.7).
    if (p.split > 1)
        p.stages = std::min(p.stages, std::max(cdiv(p.blocks, p.split),
                                               cdiv(static_cast<long long>(std::min(p.n, N)) * 512, F::kStage)));
    CUtensorMap mx, mw;
    cudaError_t e = make_byte_map(&mx, xq, p.n, k, ldx, N);
    if (e == cudaSuccess) e = make_byte_map(&mw, wq, p.m, k, ldw, 128);
    if (e != cudaSuccess) return e;
    static std::atomic<unsigned long long> allowed{0};
    const int grid = static_cast<int>(p.split > 1 ? tiles * p.split : std::min<long long>(tiles, num_sms));
    // Shared memory in proportion to the TMEM columns, so that no mix of CTAs on an SM asks for more than its 512: a
    // CTA that waits for columns while its cluster's others hold some could otherwise wait for a cluster that waits
    // for it.  (An SM has 228 KB, each CTA 1 KB of its own.)
    const int share = static_cast<int>(233472ll * F::kColumns / 512) - 1024;
    return launch_linear(linear_fp8_few_kernel<N, T>, allowed, mx, mw, p, grid, F::kThreads, p.split,
                         std::max(share, p.stages * F::kStage + F::kScaleBytes + kBarBytes + 1024), s);
}

template <typename T>
cudaError_t launch_tokens(LinearParams& p, const uint8_t* xq, size_t ldx, const uint8_t* wq, size_t ldw, int k, int num_sms,
                          cudaStream_t s) {
    const int n = p.n, m = p.m;
    // One memory round trip through registers, or TMA, tcgen05 and (split) a cluster's exchange: 8 tokens take 4.2 us
    // against 5.7 for 4608 x 1536 weights (7.1 MB), 7.0 against 5.6 for 8192 x 1536 (12.6 MB); 16 tokens would take
    // 6.3 against 5.9 and 11.0 against 5.9.
    if (n <= kStreamTokens && static_cast<long long>(m) * k <= kStreamBytes) {
        const StreamParams sp{xq, wq, ldx, ldw, p.xs, p.ws, p.bias, p.y, p.mode, n, m, k, p.blocks};
        return launch_stream<T>(sp, num_sms, s);
    }
    if (n <= 16) return launch_features_on_lanes<16, T>(p, xq, ldx, wq, ldw, k, num_sms, s);
    if (n <= 32) return launch_features_on_lanes<32, T>(p, xq, ldx, wq, ldw, k, num_sms, s);
    if (n <= 64) return launch_features_on_lanes<64, T>(p, xq, ldx, wq, ldw, k, num_sms, s);
    // Rounds of K-blocks either tiling takes: a K-block costs about the same
    // time in both, a pair's covers four times the outputs.
    const long long t1 = static_cast<long long>(cdiv(n, 128)) * cdiv(m, 128);
    const long long t2 = static_cast<long long>(cdiv(n, 256)) * cdiv(m, 256);
    if (t1 > 0x3fffffffll) return cudaErrorInvalidValue;
    const int split = few_split<128, T>(t1, p.blocks, num_sms);
    const long long rounds1 = static_cast<long long>(cdiv(t1 * split, num_sms)) * cdiv(p.blocks, split);
    const long long rounds2 = static_cast<long long>(cdiv(t2, num_sms / 2)) * p.blocks;
    if (n <= 128 || rounds1 <= rounds2) return launch_features_on_lanes<128, T>(p, xq, ldx, wq, ldw, k, num_sms, s);
    p.tiles_n = cdiv(n, 256);
    p.tiles_m = cdiv(m, 256);
    p.split = 1;
    p.stages = std::min(kMaxStages, (kSmemLimit - 1024 - kBarBytes - Pair::kStoreBytes) / Pair::kStage);
    CUtensorMap mx, mw;
    cudaError_t e = make_byte_map(&mx, xq, n, k, ldx, 128);
    if (e == cudaSuccess) e = make_byte_map(&mw, wq, m, k, ldw, 128);
    if (e != cudaSuccess) return e;
    const int grid = 2 * static_cast<int>(std::min<long long>(t2, num_sms / 2));
    if (p.mode == kGemvSwiGLU) return launch_pairs<T, kGemvSwiGLU>(mx, mw, p, grid, s);
    if (p.mode == kGemvResidual) return launch_pairs<T, kGemvResidual>(mx, mw, p, grid, s);
    return launch_pairs<T, kGemvPlain>(mx, mw, p, grid, s);
}

}  // namespace

cudaError_t launch_linear_fp8(int mode, int dtype, const uint8_t* xq, size_t ldx, const float* xs, const uint8_t* wq,
                              size_t ldw, const float* ws, const float* bias, void* y, int n, int m, int k, int num_sms,
                              cudaStream_t s) {
    LinearParams p{};
    p.xs = xs, p.ws = ws, p.bias = bias, p.y = y;
    p.mode = mode, p.n = n, p.m = m, p.blocks = cdiv(k, kFp8Block);
    switch (dtype) {
        case kF32: return launch_tokens<float>(p, xq, ldx, wq, ldw, k, num_sms, s);
        case kBF16: return launch_tokens<__nv_bfloat16>(p, xq, ldx, wq, ldw, k, num_sms, s);
        case kF16: return launch_tokens<__half>(p, xq, ldx, wq, ldw, k, num_sms, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace xl
