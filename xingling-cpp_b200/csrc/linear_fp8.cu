// Matrix product in e4m3 with a scale for each block of 128, on tcgen05.
//
//   Y[i][j] = sum_b sx[i][b] sw[j / 128][b] sum_{c in block b} xq[i][c] wq[j][c] + bias[j]
//
// A K-block is one scale block: 128 columns = 128 bytes, the SWIZZLE_128B span.
// Tokens are the MMA's M (TMEM lanes), features its N (TMEM columns): a thread
// of the epilogue then holds one token, for which sx sw is one number for all
// features of a 128-block, so scaling a K-block's sum into the fp32 result is
// one multiply-add per value with no loads.  The tensor core sums within a
// block (products of e4m3 values are exact in fp32), registers across blocks.
//
// One warp issues TMA loads into a ring of stages, one thread the MMAs of a
// K-block into the next of several TMEM accumulators, 4 or 8 warps drain
// them; the accumulators decouple the two, so the tensor core only waits for
// operands.
//
// Two tilings:
//   * 128 tokens x 128 features on one SM; fewer tiles than SMs split K over
//     the CTAs of a cluster, whose partial tiles meet in distributed shared
//     memory, each CTA finishing a share of the columns (a fixed order of
//     sums, no workspace).  Few tokens load few rows: the rest of the A tile
//     is whatever the stage holds, and only its own (unread) lanes see it.
//   * 256 x 256 on two SMs (cta_group::2), each with half of either operand:
//     64 bytes a clock from L2 per SM where a 128 x 256 tile on one SM needs
//     96, twice the reuse of the 128 x 128 tile.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fp8.cuh"
#include "tcgen05.cuh"
#include "xl_device.cuh"
#include "xl_kernels.h"

namespace xl {

namespace {

constexpr int kRows = 128;                   // token rows of a CTA's A tile
constexpr int kOpBytes = 128 * kFp8Block;    // 16 KB: 128 rows of a K-block
constexpr int kMaxStages = 12;
constexpr int kMaxSplit = 8;                 // portable cluster size
constexpr int kStagePitch = 20;              // floats a row of the store staging: 16 and padding, conflict-free in float4
constexpr int kSmemLimit = 232448;           // 227 KB
constexpr int kBarBytes = 512;
constexpr int kPartPitch = kRows + 1;        // split: partial tile [128 features][129]

template <int CG>
struct Tile {
    static constexpr int kTokens = CG * kRows;          // of the tile, all CTAs
    static constexpr int kFeatures = CG * 128;          // each CTA loads 128 of them
    static constexpr int kEpiWarps = 4 * CG;            // each drains 32 lanes x 128 columns
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kAccs = 512 / kFeatures;       // TMEM accumulators
    static constexpr int kStoreBytes = kEpiWarps * 32 * kStagePitch * 4;
    // kind::f8f6f4, e4m3 x e4m3, fp32 sums, K-major operands
    static constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(kFeatures >> 3) << 17) |
                                       (static_cast<uint32_t>(kTokens >> 4) << 24);
};

struct LinearParams {
    const float *xs, *ws, *bias;
    void* y;
    int mode, n, m, blocks;     // blocks: K-blocks
    int x_rows;                 // token rows a CTA loads (a multiple of 8, at most 128)
    int stages, stage_bytes;
    int split;                  // CTAs of a cluster that share a tile's K-blocks (one-SM tiling)
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

// 16 columns of the warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
// The loads so far have landed; naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
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

template <typename T>
__device__ __forceinline__ void put(T* dst, float v, int mode) {
    *dst = from_float<T>(mode == kGemvResidual ? to_float(*dst) + v : v);
}

// 32 tokens x 128 features in registers (a token a lane) to y, 16 outputs a
// row at a time through the warp's staging rows, so that stores are 16 bytes
// a lane along the rows.
template <typename T>
__device__ __forceinline__ void store_rows(const unsigned long long (&acc)[64], const LinearParams& p, int tok0, int j0,
                                           float* st, int lane) {
    const int wide = p.mode == kGemvSwiGLU ? p.m / 2 : p.m;
    const bool vec = (static_cast<size_t>(wide) * sizeof(T)) % 16 == 0;
    T* y = static_cast<T*>(p.y);
    constexpr int kPer = 16 / sizeof(T);  // outputs of a 16-byte store
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
        int o0 = j0 + ch * 16;
        if (p.mode == kGemvSwiGLU) {
            if (ch >= 4) break;
            o0 = j0 / 2 + ch * 16;
        }
        if (o0 >= wide) break;
        float v[16];
        if (p.mode == kGemvSwiGLU) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 ac = unpack2(acc[((ch & 3) * 16 + i)]);
                const int j = j0 + (ch & 3) * 32 + 2 * i;
                const bool on = p.bias && j < p.m;
                const float a = ac.x + (on ? p.bias[j] : 0.0f), c = ac.y + (on ? p.bias[j + 1] : 0.0f);
                v[i] = silu(a) * c;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 a = unpack2(acc[ch * 8 + i]);
                const int j = o0 + 2 * i;
                v[2 * i] = a.x + (p.bias && j < p.m ? p.bias[j] : 0.0f);
                v[2 * i + 1] = a.y + (p.bias && j + 1 < p.m ? p.bias[j + 1] : 0.0f);
            }
        }
        float4* row = reinterpret_cast<float4*>(st + lane * kStagePitch);
#pragma unroll
        for (int i = 0; i < 4; ++i) row[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        __syncwarp();
        if (vec && o0 + 16 <= wide) {
            constexpr int kLanes = 16 / kPer;  // lanes a row
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 32 / kLanes) {
                const int r = r0 + lane / kLanes, c = lane % kLanes * kPer;
                if (tok0 + r < p.n) {
                    const float* src = st + r * kStagePitch + c;
                    T* dst = y + static_cast<size_t>(tok0 + r) * wide + o0 + c;
                    uint4 out;
                    T* e = reinterpret_cast<T*>(&out);
                    if (p.mode == kGemvResidual) {
                        out = *reinterpret_cast<const uint4*>(dst);
#pragma unroll
                        for (int i = 0; i < kPer; ++i) e[i] = from_float<T>(to_float(e[i]) + src[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < kPer; ++i) e[i] = from_float<T>(src[i]);
                    }
                    *reinterpret_cast<uint4*>(dst) = out;
                }
            }
        } else {
#pragma unroll 1
            for (int r0 = 0; r0 < 32; r0 += 2) {
                const int r = r0 + lane / 16, c = lane % 16;
                if (tok0 + r < p.n && o0 + c < wide)
                    put(y + static_cast<size_t>(tok0 + r) * wide + o0 + c, st[r * kStagePitch + c], p.mode);
            }
        }
        __syncwarp();
    }
}

template <int CG, typename T>
__global__ void __launch_bounds__(Tile<CG>::kThreads, 1)
    linear_fp8_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                      const LinearParams p) {
    using TL = Tile<CG>;
    extern __shared__ __align__(1024) char smem_raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* store = reinterpret_cast<float*>(ring + p.stages * p.stage_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(store) + TL::kStoreBytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* done = empty + kMaxStages;  // an accumulator holds a K-block's sums
    uint64_t* freed = done + TL::kAccs;   // its columns have been read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(freed + TL::kAccs);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 || p.split > 1 ? cluster_rank() : 0u;
    const int group = CG == 2 ? 2 : p.split;  // CTAs that share a tile
    const int unit = static_cast<int>(blockIdx.x) / group, units = static_cast<int>(gridDim.x) / group;
    const int tiles = p.tiles_n * p.tiles_m;
    const int kb0 = CG == 2 ? 0 : static_cast<int>(static_cast<long long>(rank) * p.blocks / p.split);
    const int kb1 = CG == 2 ? p.blocks : static_cast<int>(static_cast<long long>(rank + 1) * p.blocks / p.split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < TL::kAccs; ++a) {
            mbar_init(&done[a], 1);
            mbar_init(&freed[a], CG * TL::kEpiWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&map_x), "l"(&map_w) : "memory");
    }
    if (warp == 1) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (CG == 2) cluster_sync();  // the peer's barriers are set up before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;

    // Token tiles advance fastest: the CTAs that run together share W tiles
    // and, over the whole product, either operand stays in L2.
    const uint32_t a_bytes = static_cast<uint32_t>(p.x_rows) * kFp8Block;
    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0, issued = 0;
            bool ok = true;
            for (int t = unit; t < tiles && ok; t += units) {
                const int tn = t % p.tiles_n, tm = t / p.tiles_n;
                const int y_x = tn * TL::kTokens + (CG == 2 ? static_cast<int>(rank) * kRows : 0);
                const int y_w = tm * TL::kFeatures + (CG == 2 ? static_cast<int>(rank) * 128 : 0);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait_bar(&empty[s], ph ^ 1u, nullptr)) {
                        ok = false;
                        break;
                    }
                    const uint32_t st = smem_u32(ring + s * p.stage_bytes);
                    uint32_t bar = smem_u32(&full[s]);
                    if (CG == 2) bar = cluster_addr(bar, 0);
                    if (CG == 1 || rank == 0) mbar_expect_tx(&full[s], CG * (a_bytes + kOpBytes));
                    load_tile<CG>(st, &map_x, kb * kFp8Block, y_x, bar);
                    load_tile<CG>(st + a_bytes, &map_w, kb * kFp8Block, y_w, bar);
                    ++issued;
                    if (++s == p.stages) s = 0, ph ^= 1u;
                }
            }
            if (!ok && (CG == 1 || rank == 0)) {
                // the copies in flight land before the CTA leaves
                for (uint32_t i = 0; i < min(issued, static_cast<uint32_t>(p.stages)); ++i) {
                    if (s == 0) s = p.stages, ph ^= 1u;
                    --s;
                    wait_bar(&full[s], ph, nullptr);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && (CG == 1 || rank == 0)) {
            int s = 0, a = 0;
            uint32_t ph = 0, pa = 0;
            bool ok = true;
            for (int t = unit; t < tiles && ok; t += units) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!wait_bar(&freed[a], pa ^ 1u, nullptr) || !wait_bar(&full[s], ph, nullptr)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t st = smem_u32(ring + s * p.stage_bytes);
                    const uint64_t da = umma_desc(st), db = umma_desc(st + a_bytes);
                    const uint32_t acc = tmem + static_cast<uint32_t>(a * TL::kFeatures);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)  // 32 columns = 32 bytes each
                        mma_e4m3<CG>(acc, da + 2 * ks, db + 2 * ks, TL::kIdesc, ks != 0);
                    commit<CG>(&empty[s]);
                    commit<CG>(&done[a]);
                    if (++s == p.stages) s = 0, ph ^= 1u;
                    if (++a == TL::kAccs) a = 0, pa ^= 1u;
                }
            }
        }
    } else {
        // TMEM lanes are a warp's by its number modulo 4
        const int q = warp & 3, half = (warp - 2) >> 2;
        float* st = store + (warp - 2) * 32 * kStagePitch;
        int a = 0;
        uint32_t pa = 0;
        bool ok = true;
        for (int t = unit; t < tiles; t += units) {
            const int tn = t % p.tiles_n, tm = t / p.tiles_n;
            const int tok0 = tn * TL::kTokens + (CG == 2 ? static_cast<int>(rank) * kRows : 0) + 32 * q;
            const int j0 = tm * TL::kFeatures + 128 * half;
            const bool work = tok0 < p.n && j0 < p.m;  // else the warp only keeps the accumulators moving
            const float* xs = p.xs + static_cast<size_t>(min(tok0 + lane, p.n - 1)) * p.blocks;
            const float* ws = p.ws + static_cast<size_t>(min(j0, p.m - 1) / kFp8Block) * p.blocks;
            unsigned long long acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            float sx = kb0 < kb1 ? xs[kb0] : 0.0f, sw = kb0 < kb1 ? ws[kb0] : 0.0f;
#pragma unroll 1
            for (int kb = kb0; kb < kb1; ++kb) {
                const float s = sx * sw;
                if (kb + 1 < kb1) sx = xs[kb + 1], sw = ws[kb + 1];
                if (ok) ok = __all_sync(0xffffffffu, wait_bar(&done[a], pa, nullptr));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (work && ok) {
                    const uint32_t ta = tmem + (static_cast<uint32_t>(32 * q) << 16) +
                                        static_cast<uint32_t>(a * TL::kFeatures + 128 * half);
                    const unsigned long long s2 = pack2(__float_as_uint(s), __float_as_uint(s));
                    uint32_t r0[16], r1[16];
                    tmem_load16(ta, r0);
#pragma unroll
                    for (int c = 0; c < 8; c += 2) {
                        tmem_wait16(r0);
                        tmem_load16(ta + 16 * (c + 1), r1);
#pragma unroll
                        for (int i = 0; i < 8; ++i) fma2(acc[c * 8 + i], pack2(r0[2 * i], r0[2 * i + 1]), s2);
                        tmem_wait16(r1);
                        if (c + 2 < 8) tmem_load16(ta + 16 * (c + 2), r0);
#pragma unroll
                        for (int i = 0; i < 8; ++i) fma2(acc[(c + 1) * 8 + i], pack2(r1[2 * i], r1[2 * i + 1]), s2);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    uint32_t bar = smem_u32(&freed[a]);
                    if (CG == 2) bar = cluster_addr(bar, 0);
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
                }
                if (++a == TL::kAccs) a = 0, pa ^= 1u;
            }
            if (!ok) {  // a wait ran out: the results say so
#pragma unroll
                for (int i = 0; i < 64; ++i) acc[i] = 0x7fffffff7fffffffull;
            }
            if (CG == 2 || p.split == 1) {
                if (work) store_rows<T>(acc, p, tok0, j0, st, lane);
            } else {
                // every K-block of this CTA has been multiplied: the ring is free for the partial tile
                float* part = reinterpret_cast<float*>(ring);
                if (work && tok0 + lane < p.n) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        const float2 v = unpack2(acc[i]);
                        part[(2 * i) * kPartPitch + 32 * q + lane] = v.x;
                        part[(2 * i + 1) * kPartPitch + 32 * q + lane] = v.y;
                    }
                }
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (CG == 1 && p.split > 1) {
        __syncwarp();
        cluster_sync();
        // A cluster has one tile; this CTA finishes 128 / split of its columns.
        const int tn = unit % p.tiles_n, tm = unit / p.tiles_n;
        const int rows = min(kRows, p.n - tn * kRows), step = p.mode == kGemvSwiGLU ? 2 : 1;
        const int cols = 128 / p.split, outs = cols / step, wide = p.m / step;
        const uint32_t part = smem_u32(ring);
        T* y = static_cast<T*>(p.y);
        for (int e = threadIdx.x; e < rows * outs; e += TL::kThreads) {
            const int r = e / outs, c = static_cast<int>(rank) * cols + (e - r * outs) * step, j = tm * 128 + c;
            if (j >= p.m) continue;
            float v[2] = {0.0f, 0.0f};
            for (int i = 0; i < step; ++i) {
                const uint32_t at = part + static_cast<uint32_t>((c + i) * kPartPitch + r) * 4;
                for (int k = 0; k < p.split; ++k) {
                    float x;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(cluster_addr(at, k)) : "memory");
                    v[i] += x;
                }
                if (p.bias) v[i] += p.bias[j + i];
            }
            put(y + static_cast<size_t>(tn * kRows + r) * wide + j / step, step == 2 ? silu(v[0]) * v[1] : v[0], p.mode);
        }
    }
    __syncwarp();
    __syncthreads();
    if (CG == 2 || p.split > 1) cluster_sync();  // no CTA leaves while another may reach its shared memory
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int CG, typename T>
cudaError_t launch_tiled(const CUtensorMap& mx, const CUtensorMap& mw, const LinearParams& p, int grid, cudaStream_t s) {
    using TL = Tile<CG>;
    const int smem = p.stages * p.stage_bytes + TL::kStoreBytes + kBarBytes + 1024;
    cudaError_t e = cudaFuncSetAttribute(linear_fp8_kernel<CG, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(TL::kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    const int cluster = CG == 2 ? 2 : p.split;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    count_launch();
    return cudaLaunchKernelEx(&cfg, linear_fp8_kernel<CG, T>, mx, mw, p);
}

int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

}  // namespace

cudaError_t launch_linear_fp8(int mode, int dtype, const uint8_t* xq, size_t ldx, const float* xs, const uint8_t* wq,
                              size_t ldw, const float* ws, const float* bias, void* y, int n, int m, int k, int num_sms,
                              cudaStream_t s) {
    LinearParams p{};
    p.xs = xs, p.ws = ws, p.bias = bias, p.y = y;
    p.mode = mode, p.n = n, p.m = m, p.blocks = cdiv(k, kFp8Block);
    // Rounds of K-blocks either tiling takes: a K-block costs about the same
    // time in both (operands from L2), a pair's covers four times the outputs.
    const long long t1 = static_cast<long long>(cdiv(n, 128)) * cdiv(m, 128);
    const long long t2 = static_cast<long long>(cdiv(n, 256)) * cdiv(m, 256);
    if (t1 > 0x3fffffffll) return cudaErrorInvalidValue;
    int split = 1;
    while (split < kMaxSplit && t1 * split * 2 <= num_sms && split * 2 <= p.blocks) split *= 2;
    const long long rounds1 = static_cast<long long>(cdiv(t1 * split, num_sms)) * cdiv(p.blocks, split);
    const long long rounds2 = static_cast<long long>(cdiv(t2, num_sms / 2)) * p.blocks;
    const bool pair = n > 128 && rounds2 < rounds1;
    p.split = pair ? 1 : split;
    p.tiles_n = cdiv(n, pair ? 256 : 128);
    p.tiles_m = cdiv(m, pair ? 256 : 128);
    p.x_rows = pair || n >= kRows ? kRows : cdiv(n, 8) * 8;
    p.stage_bytes = p.x_rows * kFp8Block + kOpBytes;
    const int room = kSmemLimit - 1024 - kBarBytes - (pair ? Tile<2>::kStoreBytes : Tile<1>::kStoreBytes);
    p.stages = std::min(kMaxStages, room / p.stage_bytes);
    CUtensorMap mx, mw;
    cudaError_t e = make_byte_map(&mx, xq, n, k, ldx, p.x_rows);
    if (e == cudaSuccess) e = make_byte_map(&mw, wq, m, k, ldw, 128);
    if (e != cudaSuccess) return e;
    const long long tiles = static_cast<long long>(p.tiles_n) * p.tiles_m;
    const int grid = pair ? 2 * static_cast<int>(std::min<long long>(tiles, num_sms / 2))
                          : p.split * static_cast<int>(p.split > 1 ? tiles : std::min<long long>(tiles, num_sms));
    auto go = [&](auto t) {
        using T = decltype(t);
        return pair ? launch_tiled<2, T>(mx, mw, p, grid, s) : launch_tiled<1, T>(mx, mw, p, grid, s);
    };
    switch (dtype) {
        case kF32: return go(float{});
        case kBF16: return go(__nv_bfloat16{});
        case kF16: return go(__half{});
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace xl
