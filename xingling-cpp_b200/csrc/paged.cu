// A paged key/value cache: append of rows, and attention of one new token per sequence.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

#include "fp8.cuh"
#include "paged.h"
#include "xl_device.cuh"
#include "xl_kernels.h"

namespace xl {

namespace {

// Rotation of the pair (a, b) = (x[j], x[j + d/2]) by the table's angle (the engine's rotate-half RoPE).
__device__ __forceinline__ void rotate(float& a, float& b, float2 cs) {
    const float x = a, y = b;
    a = x * cs.x + y * cs.y;
    b = y * cs.x - x * cs.y;
}

// 16 elements a thread: of a key 8 pairs (j, j + d/2), of a value 16 in a row.
template <typename T, typename C>
__global__ void __launch_bounds__(256) kv_append_paged_kernel(const PagedCache pc, const T* __restrict__ qkv,
                                                              const float2* __restrict__ rope, int rope_len,
                                                              const int* __restrict__ row_seq,
                                                              const int* __restrict__ row_pos, int rows, int heads) {
    const int d = pc.head_dim, per_head = d / 16, per_side = pc.kv_heads * per_head;
    const long long id = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    const int row = static_cast<int>(id / (2 * per_side));
    if (row >= rows) return;
    const int rest = static_cast<int>(id - static_cast<long long>(row) * (2 * per_side));
    const bool value = rest >= per_side;
    const int h = (value ? rest - per_side : rest) / per_head, part = (value ? rest - per_side : rest) % per_head;
    const int seq = row_seq[row], pos = row_pos[row];
    if (seq < 0 || seq >= pc.batch || !paged_pos_ok(pos, pc.max_pages, pc.page_size, rope ? rope_len : 0)) return;
    const int page = pc.page_table[static_cast<int64_t>(seq) * pc.max_pages + pos / pc.page_size];
    if (!paged_valid(page, pc.num_pages)) return;
    const int64_t at = paged_base(page, h, pc.kv_heads, pc.page_size, d) + static_cast<int64_t>(pos % pc.page_size) * d;
    const T* src = qkv + static_cast<int64_t>(row) * (heads + 2 * pc.kv_heads) * d +
                   static_cast<int64_t>(heads + (value ? pc.kv_heads : 0) + h) * d;
    const int e0 = value ? part * 16 : part * 8, e1 = value ? e0 + 8 : e0 + d / 2;
    float a[8], b[8];
    load8(src + e0, a);
    load8(src + e1, b);
    if (!value && rope) {
#pragma unroll
        for (int i = 0; i < 8; ++i) rotate(a[i], b[i], rope[static_cast<int64_t>(pos) * (d / 2) + e0 + i]);
    }
    C* dst = static_cast<C*>(value ? pc.v : pc.k) + at;
    store8(dst + e0, a);
    store8(dst + e1, b);
}

// ---- attention of one new token a sequence ------------------------------------------------------------------------
//
//   o = sum_t w_t v_t / sum_t w_t,  w_t = exp(q . k_t / sqrt(d)),  t = 0 .. pos
//
// One pass over the cache with the running maximum and sum of a softmax.  What
// bounds it is reading the cache, so the work is cut by cache bytes: every
// (sequence, key/value head, block of 8 or 16 query heads) is a "pair" of
// chunks of 4 x kTile positions, the chunks of all pairs stand in one row, and
// every CTA takes an equal stretch of that row (lengths live on the device; a
// CTA finds its stretch from them).  A pair that one CTA covers is finished
// there; else its CTAs leave (maximum, sum, output) partials in the workspace
// and the last to arrive (a ticket, nobody waits) merges them in CTA order, so
// results do not depend on timing.
//
// Within a CTA each warp takes tiles of kTile positions with its own running
// softmax.  Query heads that share a key/value head are the rows of
// mma.sync tiles, so a byte of cache is read once for all of them and turned
// into scores without shuffles.  The cache goes from global memory straight
// into the MMA's register layout, 16 bytes a load: the columns that a lane
// holds are a permutation of the MMA's, applied alike to both operands of the
// scores (any order of d sums the same) and, for the values, undone when the
// output is stored.
//
// Precision: queries are split in two 16-bit halves (scaled by a power of two
// so that they fit fp16), and so are the weights, which leaves 2^-17 of error
// where rounding them would leave 2^-9; an fp32 cache runs as three TF32
// products of split operands.  Sums, maxima and the running output are fp32.

constexpr int kAttnWarps = 4;
constexpr int kAttnMaxCtas = 592;            // 148 SMs x 4
constexpr int kAttnRows = 16;                // most query heads of a pair
constexpr size_t kAttnSlotFloats = kAttnRows * (128 + 2);
constexpr size_t kAttnPartBytes = kAttnMaxCtas * 2 * kAttnSlotFloats * 4;  // two partials a CTA
constexpr uint32_t kNoRow = 0xffffffffu;     // masked or unreadable: zeros
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
    PagedCache pc;
    const void* qkv;
    const float2* rope;
    int rope_len;
    const int* pos;
    void* out;
    int heads, group, blocks;  // query heads a key/value head has; pairs (blocks of heads) a key/value head has
    int io;                    // DType of qkv and out
    FastDiv page_div;
    float* part;               // [grid][2][rows][d + 2]
    int* tickets;              // [batch][kv_heads][blocks], zero between calls
};

__device__ __forceinline__ float load_io(const void* p, int64_t i, int io) {
    if (io == kF32) return static_cast<const float*>(p)[i];
    if (io == kBF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_io(void* p, int64_t i, float v, int io) {
    if (io == kF32) static_cast<float*>(p)[i] = v;
    else if (io == kBF16) static_cast<__nv_bfloat16*>(p)[i] = from_float<__nv_bfloat16>(v);
    else static_cast<__half*>(p)[i] = from_float<__half>(v);
}

__device__ __forceinline__ uint32_t pack16(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Two values as a pair of 16-bit halves: v = hi + lo up to 2^-17 (bf16) or 2^-22 (fp16) of it.
template <typename C>
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ha = to_float(from_float<C>(a)), hb = to_float(from_float<C>(b));
    hi = pack16(ha, hb, C{});
    lo = pack16(a - ha, b - hb, C{});
}
__device__ __forceinline__ uint32_t tf32_lo(uint32_t v) {
    return __float_as_uint(__uint_as_float(v) - __uint_as_float(v & 0xffffe000u));
}

__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two products of a split value with an unsplit one (16-bit caches).
template <typename C>
__device__ __forceinline__ void mma_split(float (&d)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], uint32_t b0,
                                          uint32_t b1) {
    mma16(d, hi, b0, b1, C{});
    mma16(d, lo, b0, b1, C{});
}
// Three TF32 products: fp32 accuracy up to the dropped lo . lo (2^-22).  The
// MMA reads the upper 19 bits of its operands, so a value is its own hi.
__device__ __forceinline__ void mma_split3(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const uint32_t lo[4] = {tf32_lo(a[0]), tf32_lo(a[1]), tf32_lo(a[2]), tf32_lo(a[3])};
    mma_tf32(d, a, b0, b1);
    mma_tf32(d, a, tf32_lo(b0), tf32_lo(b1));
    mma_tf32(d, lo, b0, b1);
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// C: cache type, D: head dim, WIDE: 16 query heads a pair (else 8, and the MMA's rows 8 .. 15 idle).
template <typename C, int D, bool WIDE>
struct AttnShape {
    static constexpr bool k32 = sizeof(C) == 4;
    static constexpr int kVec = 16 / sizeof(C);             // elements of a 16-byte load
    static constexpr int kNT = k32 && D == 128 ? 1 : 2;     // 8-position MMA tiles of a warp tile
    static constexpr int kTile = 8 * kNT;
    static constexpr int kChunk = kAttnWarps * kTile;
    static constexpr int kKch = D / (4 * kVec);             // 16-byte loads of a lane per key row
    static constexpr int kVch = D / (8 * kVec);             // ... per value row
    static constexpr int kSteps = 2 * kKch;                 // MMA steps of a score
    static constexpr int kRows = WIDE ? 16 : 8;
    static constexpr int kQPitch = D + 4;
    static constexpr int kSmemFloats = kRows * kQPitch + kAttnWarps * kRows * (D + 2);
    static constexpr int kCtas = WIDE ? 2 : 3;              // an SM holds, by registers
};

template <typename C, int D, bool WIDE>
__global__ void __launch_bounds__(128, (AttnShape<C, D, WIDE>::kCtas)) attn_decode_paged_kernel(const AttnParams p) {
    using S = AttnShape<C, D, WIDE>;
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;                              // [rows][D + 4] rotated queries
    float* warp_part = smem + S::kRows * S::kQPitch;  // [warps][rows][D + 2]
    __shared__ int flag;
    const PagedCache& pc = p.pc;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pairs = pc.kv_heads * p.blocks;  // of a sequence
    const int64_t width = static_cast<int64_t>(p.heads + 2 * pc.kv_heads) * D;
    C *kp = static_cast<C*>(pc.k), *vp = static_cast<C*>(pc.v);
    const int limit = p.rope ? p.rope_len : 0;

    auto chunks_of = [&](int pos) {
        return paged_pos_ok(pos, pc.max_pages, pc.page_size, limit) ? pos / S::kChunk + 1 : 1;
    };
    // Every warp adds up all sequences' chunks, then finds the sequence its CTA's stretch begins in.
    long long total = 0;
    for (int b0 = 0; b0 < pc.batch; b0 += 32) {
        long long c = b0 + lane < pc.batch ? chunks_of(p.pos[b0 + lane]) : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
        total += c;
    }
    const long long all = total * pairs;
    const long long grid = min(static_cast<long long>(gridDim.x), all);  // a chunk at least for every CTA that works
    if (blockIdx.x >= grid) return;
    long long at = blockIdx.x * all / grid;
    const long long end = (blockIdx.x + 1) * all / grid;
    int b = 0;
    long long first = 0;  // the row's index of sequence b's first chunk
    for (int b0 = 0; b0 < pc.batch; b0 += 32) {
        const long long own = b0 + lane < pc.batch ? chunks_of(p.pos[b0 + lane]) * static_cast<long long>(pairs) : 0;
        long long upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, first + upto > at);
        if (past) {
            const int i = __ffs(past) - 1;
            b = b0 + i;
            first += __shfl_sync(0xffffffffu, upto - own, i);
            break;
        }
        first += __shfl_sync(0xffffffffu, upto, 31);
    }

    while (at < end) {
        const int pos = p.pos[b];
        const int nch = chunks_of(pos);
        const int pair = static_cast<int>((at - first) / nch);
        const int c0 = static_cast<int>((at - first) - static_cast<long long>(pair) * nch);
        const int c1 = static_cast<int>(min(static_cast<long long>(nch), c0 + (end - at)));
        const int kh = pair / p.blocks, blk = pair - kh * p.blocks;
        const int h0 = kh * p.group + blk * S::kRows, nh = min(S::kRows, p.group - blk * S::kRows);
        const int64_t out0 = (static_cast<int64_t>(b) * p.heads + h0) * D;
        const long long pair_first = first + static_cast<long long>(pair) * nch;
        at += c1 - c0;
        if (pair == pairs - 1 && c1 == nch) {
            first += static_cast<long long>(pairs) * nch;
            ++b;
        }
        const int seq = pair == pairs - 1 && c1 == nch ? b - 1 : b;
        if (!paged_pos_ok(pos, pc.max_pages, pc.page_size, limit)) {
            const float v = pos == -1 ? 0.0f : __int_as_float(0x7fffffff);
            for (int i = threadIdx.x; i < nh * D; i += 128) store_io(p.out, out0 + i, v, p.io);
            continue;
        }
        const int* table = pc.page_table + static_cast<int64_t>(seq) * pc.max_pages;
        const int64_t qrow = seq * width;

        // The rotated queries, and in the CTA that holds the last position its new key and value.
        __syncthreads();  // the last pair's shared memory has been read
        for (int i = threadIdx.x; i < S::kRows * (D / 2); i += 128) {
            const int r = i / (D / 2), j = i - r * (D / 2);
            float a = 0.0f, c = 0.0f;
            if (r < nh) {
                const int64_t src = qrow + static_cast<int64_t>(h0 + r) * D + j;
                a = load_io(p.qkv, src, p.io), c = load_io(p.qkv, src + D / 2, p.io);
                if (p.rope) rotate(a, c, p.rope[static_cast<int64_t>(pos) * (D / 2) + j]);
            }
            qs[r * S::kQPitch + j] = a;
            qs[r * S::kQPitch + j + D / 2] = c;
        }
        if (c1 == nch) {
            const int page = table[p.page_div.div(pos)];
            if (paged_valid(page, pc.num_pages) && threadIdx.x < D / 2) {
                const int j = threadIdx.x;
                const int64_t dst = paged_base(page, kh, pc.kv_heads, pc.page_size, D) +
                                    static_cast<int64_t>(pos - p.page_div.div(pos) * pc.page_size) * D + j;
                const int64_t src = qrow + static_cast<int64_t>(p.heads + kh) * D + j, sv = src + static_cast<int64_t>(pc.kv_heads) * D;
                float a = load_io(p.qkv, src, p.io), c = load_io(p.qkv, src + D / 2, p.io);
                if (p.rope) rotate(a, c, p.rope[static_cast<int64_t>(pos) * (D / 2) + j]);
                kp[dst] = from_float<C>(a), kp[dst + D / 2] = from_float<C>(c);
                vp[dst] = from_float<C>(load_io(p.qkv, sv, p.io));
                vp[dst + D / 2] = from_float<C>(load_io(p.qkv, sv + D / 2, p.io));
            }
        }
        __syncthreads();  // queries, and the new rows, are there for every warp

        // A lane's part of query rows g and g + 8, scaled to [1, 2) by a power of two.
        float back[2];  // 2^e log2(e) / sqrt(D): turns a row's products into log2 of its weights
        uint32_t qh[S::kSteps][4], ql[S::k32 ? 1 : S::kSteps][4];  // fp32: the values themselves
        {
            float big[2] = {0.0f, 0.0f};
#pragma unroll
            for (int r = 0; r < (WIDE ? 2 : 1); ++r) {
#pragma unroll
                for (int j = 0; j < S::kKch; ++j)
#pragma unroll
                    for (int i = 0; i < S::kVec; ++i)
                        big[r] = fmaxf(big[r], fabsf(qs[(g + 8 * r) * S::kQPitch + (4 * j + t) * S::kVec + i]));
                big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 1));
                big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 2));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int e = big[r] > 0.0f && big[r] < 3e38f ? max(-120, min(120, ilogbf(big[r]))) : 0;
                const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                back[r] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * (kLog2e / (D == 64 ? 8.0f : 11.313708498984761f));
                const float* src = qs + (g + 8 * r) * S::kQPitch;
#pragma unroll
                for (int s = 0; s < S::kSteps; ++s) {
                    const int e0 = (4 * (s / 2) + t) * S::kVec + (s & 1) * (S::kVec / 2);
                    if (!WIDE && r == 1) {
                        qh[s][1] = qh[s][3] = 0u;
                        if constexpr (!S::k32) ql[s][1] = ql[s][3] = 0u;
                    } else if constexpr (S::k32) {
                        qh[s][r] = __float_as_uint(src[e0] * down);
                        qh[s][2 + r] = __float_as_uint(src[e0 + 1] * down);
                    } else {
                        split16<C>(src[e0] * down, src[e0 + 1] * down, qh[s][r], ql[s][r]);
                        split16<C>(src[e0 + 2] * down, src[e0 + 3] * down, qh[s][2 + r], ql[s][2 + r]);
                    }
                }
            }
        }

        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
        constexpr int kAcc = WIDE ? 4 : 2;  // of an MMA's four results; rows 8 .. 15 are zeros that nobody keeps
        float acc[D / 8][kAcc];
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int j = 0; j < kAcc; ++j) acc[i][j] = 0.0f;
        bool bad = false;

        // Rows of the pool that a tile's positions are in, a position a lane.
        auto find_rows = [&](int c) {
            const int x = c * S::kChunk + warp * S::kTile + (lane & (S::kTile - 1));
            if (c >= c1 || x > pos) return kNoRow;
            const int n = static_cast<int>(p.page_div.div(x));
            const int page = table[n];
            if (!paged_valid(page, pc.num_pages)) {
                bad = true;
                return kNoRow;
            }
            return static_cast<uint32_t>((static_cast<int64_t>(page) * pc.kv_heads + kh) * pc.page_size + (x - n * pc.page_size));
        };
        uint4 kr[S::kNT][S::kKch], vr[2 * S::kNT][S::kVch];
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        auto load_k = [&](uint32_t rows) {
#pragma unroll
            for (int n = 0; n < S::kNT; ++n) {
                const uint32_t r = __shfl_sync(0xffffffffu, rows, 8 * n + g);
                const uint4* src = reinterpret_cast<const uint4*>(kp + static_cast<int64_t>(r) * D) + t;
#pragma unroll
                for (int j = 0; j < S::kKch; ++j) kr[n][j] = r == kNoRow ? zero : __ldcg(src + 4 * j);
            }
        };
        auto load_v = [&](uint32_t rows) {
#pragma unroll
            for (int n = 0; n < 2 * S::kNT; ++n) {
                const uint32_t r = __shfl_sync(0xffffffffu, rows, 8 * (n >> 1) + 2 * t + (n & 1));
                const uint4* src = reinterpret_cast<const uint4*>(vp + static_cast<int64_t>(r) * D) + g;
#pragma unroll
                for (int j = 0; j < S::kVch; ++j) vr[n][j] = r == kNoRow ? zero : __ldcg(src + 8 * j);
            }
        };
        uint32_t rows = find_rows(c0);
        load_k(rows);
        load_v(rows);
        for (int c = c0; c < c1; ++c) {
            const int x0 = c * S::kChunk + warp * S::kTile;
            const uint32_t next = find_rows(c + 1);
            if (x0 > pos) break;  // only the last chunk has tiles past the end
            float s[S::kNT][4];
#pragma unroll
            for (int n = 0; n < S::kNT; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    const uint32_t b0 = word(kr[n][i / 2], (i & 1) * 2), b1 = word(kr[n][i / 2], (i & 1) * 2 + 1);
                    if constexpr (S::k32) mma_split3(s[n], qh[i], b0, b1);
                    else mma_split<C>(s[n], qh[i], ql[i], b0, b1);
                }
            }
            load_k(next);
            float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < S::kNT; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[n][j] = x0 + 8 * n + 2 * t + (j & 1) <= pos ? s[n][j] * back[j >> 1] : -INFINITY;
                    if (WIDE || j < 2) high[j >> 1] = fmaxf(high[j >> 1], s[n][j]);
                }
            float old[2] = {1.0f, 1.0f};
#pragma unroll
            for (int r = 0; r < (WIDE ? 2 : 1); ++r) {
                high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 1));
                high[r] = fmaxf(high[r], __shfl_xor_sync(0xffffffffu, high[r], 2));
                high[r] = fmaxf(high[r], top[r]);
                old[r] = exp2f(top[r] - high[r]);
                top[r] = high[r];
                sum[r] *= old[r];
            }
            if (__any_sync(0xffffffffu, old[0] != 1.0f || old[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
#pragma unroll
                    for (int j = 0; j < kAcc; ++j) acc[i][j] *= old[j >> 1];
            }
            uint32_t wh[S::kNT][4], wl[S::kNT][4];
#pragma unroll
            for (int n = 0; n < S::kNT; ++n) {
#pragma unroll
                for (int j = 0; j < (WIDE ? 4 : 2); ++j) {
                    s[n][j] = exp2f(s[n][j] - top[j >> 1]);
                    sum[j >> 1] += s[n][j];
                }
                if (!WIDE) s[n][2] = s[n][3] = 0.0f;
            }
            if constexpr (S::k32) {
                // position 2t is the MMA's k = t, 2t + 1 its k = t + 4
#pragma unroll
                for (int n = 0; n < S::kNT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        wh[n][j] = __float_as_uint(s[n][(j & 1) * 2 + (j >> 1)]);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    float o[4] = {acc[i][0], acc[i][1], WIDE ? acc[i][kAcc - 2] : 0.0f, WIDE ? acc[i][kAcc - 1] : 0.0f};
#pragma unroll
                    for (int n = 0; n < S::kNT; ++n)
                        mma_split3(o, wh[n], word(vr[2 * n][i / S::kVec], i % S::kVec),
                                   word(vr[2 * n + 1][i / S::kVec], i % S::kVec));
#pragma unroll
                    for (int j = 0; j < kAcc; ++j) acc[i][j] = o[j];
                }
            } else {
                split16<C>(s[0][0], s[0][1], wh[0][0], wl[0][0]);
                split16<C>(s[0][2], s[0][3], wh[0][1], wl[0][1]);
                split16<C>(s[S::kNT - 1][0], s[S::kNT - 1][1], wh[0][2], wl[0][2]);
                split16<C>(s[S::kNT - 1][2], s[S::kNT - 1][3], wh[0][3], wl[0][3]);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const int ch = i / S::kVec, e = i % S::kVec;
                    const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;
                    const uint32_t b0 = __byte_perm(word(vr[0][ch], e / 2), word(vr[1][ch], e / 2), pick);
                    const uint32_t b1 = __byte_perm(word(vr[2 * S::kNT - 2][ch], e / 2), word(vr[2 * S::kNT - 1][ch], e / 2), pick);
                    float o[4] = {acc[i][0], acc[i][1], WIDE ? acc[i][kAcc - 2] : 0.0f, WIDE ? acc[i][kAcc - 1] : 0.0f};
                    mma_split<C>(o, wh[0], wl[0], b0, b1);
#pragma unroll
                    for (int j = 0; j < kAcc; ++j) acc[i][j] = o[j];
                }
            }
            load_v(next);
        }

        // The warps' rows: output parts, then maximum and sum.
#pragma unroll
        for (int r = 0; r < (WIDE ? 2 : 1); ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            float* row = warp_part + (warp * S::kRows + g + 8 * r) * (D + 2);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                const int d = (i / S::kVec) * 8 * S::kVec + 2 * t * S::kVec + i % S::kVec;
                row[d] = acc[i][(2 * r) % kAcc];
                row[d + S::kVec] = acc[i][(2 * r + 1) % kAcc];
            }
            if (__any_sync(0xffffffffu, bad)) sum[r] = __int_as_float(0x7fffffff);
            if (t == 0) row[D] = top[r], row[D + 1] = sum[r];
        }
        __syncthreads();
        const bool whole = c0 == 0 && c1 == nch;
        const int slot = 2 * blockIdx.x + (c0 > 0 ? 0 : 1);
        float* mine = p.part + slot * static_cast<int64_t>(S::kRows * (D + 2));
        for (int i = threadIdx.x; i < nh * D; i += 128) {
            const int r = i / D, d = i - r * D;
            const float* row = warp_part + r * (D + 2);
            float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, row[w * S::kRows * (D + 2) + D]);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float* x = row + w * S::kRows * (D + 2);
                const float f = x[D] == -INFINITY ? 0.0f : exp2f(x[D] - m);
                l += f * x[D + 1], o += f * x[d];
                if (x[D + 1] != x[D + 1]) l = x[D + 1];
            }
            if (whole) {
                store_io(p.out, out0 + i, o / l, p.io);
            } else {
                mine[r * (D + 2) + d] = o;
                if (d == 0) mine[r * (D + 2) + D] = m, mine[r * (D + 2) + D + 1] = l;
            }
        }
        if (whole) continue;

        // The pair's last CTA to come here merges all its partials, in CTA order.
        const int cta0 = static_cast<int>(((pair_first + 1) * grid - 1) / all);
        const int cta1 = static_cast<int>(((pair_first + nch) * grid - 1) / all);
        int* ticket = p.tickets + static_cast<int64_t>(seq) * pairs + pair;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) flag = atomicAdd(ticket, 1) == cta1 - cta0;
        __syncthreads();
        if (!flag) continue;
        __threadfence();
        for (int i = threadIdx.x; i < nh * D; i += 128) {
            const int r = i / D, d = i - r * D;
            float m = -INFINITY, l = 0.0f, o = 0.0f;
            for (int c = cta0; c <= cta1; ++c) {
                // a pair begins within its first CTA's stretch unless that stretch begins with it
                const int sl = 2 * c + (c == cta0 ? 1 : 0);
                const float* x = p.part + sl * static_cast<int64_t>(S::kRows * (D + 2)) + r * (D + 2);
                const float xm = __ldcg(x + D), xl = __ldcg(x + D + 1), xo = __ldcg(x + d);
                const float up = fmaxf(m, xm);
                const float f0 = m == -INFINITY ? 0.0f : exp2f(m - up), f1 = xm == -INFINITY ? 0.0f : exp2f(xm - up);
                l = l * f0 + xl * f1;
                if (xl != xl) l = xl;
                o = o * f0 + xo * f1;
                m = up;
            }
            store_io(p.out, out0 + i, o / l, p.io);
        }
        if (threadIdx.x == 0) *ticket = 0;
    }
}

template <typename T, typename C>
cudaError_t append_typed(const PagedCache& pc, const void* qkv, const float* rope, int rope_len, const int* row_seq,
                         const int* row_pos, int rows, int heads, cudaStream_t s) {
    const long long items = static_cast<long long>(rows) * pc.kv_heads * (pc.head_dim / 8);
    const long long ctas = (items + 255) / 256;
    if (ctas > 0x7fffffffll) return cudaErrorInvalidValue;
    count_launch();
    kv_append_paged_kernel<T, C><<<static_cast<int>(ctas), 256, 0, s>>>(
        pc, static_cast<const T*>(qkv), reinterpret_cast<const float2*>(rope), rope_len, row_seq, row_pos, rows, heads);
    return cudaGetLastError();
}

template <typename C, int D, bool WIDE>
cudaError_t attend_shape(AttnParams p, int num_sms, cudaStream_t s) {
    using S = AttnShape<C, D, WIDE>;
    p.blocks = (p.group - 1) / S::kRows + 1;
    const long long longest = static_cast<long long>(p.pc.max_pages) * p.pc.page_size;
    const long long chunks = ((longest - 1) / S::kChunk + 1) * p.pc.batch * p.pc.kv_heads * p.blocks;
    const long long most = std::min(num_sms * S::kCtas, kAttnMaxCtas);
    count_launch();
    attn_decode_paged_kernel<C, D, WIDE>
        <<<static_cast<int>(std::min(chunks, most)), 128, S::kSmemFloats * sizeof(float), s>>>(p);
    return cudaGetLastError();
}

template <typename C>
cudaError_t attend_typed(const AttnParams& p, int num_sms, cudaStream_t s) {
    const bool wide = p.group > 8;
    if (p.pc.head_dim == 64)
        return wide ? attend_shape<C, 64, true>(p, num_sms, s) : attend_shape<C, 64, false>(p, num_sms, s);
    return wide ? attend_shape<C, 128, true>(p, num_sms, s) : attend_shape<C, 128, false>(p, num_sms, s);
}

// f(T{}, C{}) for the types of the rows and of the cache.
template <typename F>
cudaError_t by_types(int dtype, int cache, F f) {
    auto inner = [&](auto t) {
        switch (cache) {
            case kF32: return f(t, float{});
            case kBF16: return f(t, __nv_bfloat16{});
            case kF16: return f(t, __half{});
            default: return cudaErrorInvalidValue;
        }
    };
    switch (dtype) {
        case kF32: return inner(float{});
        case kBF16: return inner(__nv_bfloat16{});
        case kF16: return inner(__half{});
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_kv_append_paged(const PagedCache& pc, int dtype, const void* qkv, const float* rope, int rope_len,
                                   const int* row_seq, const int* row_pos, int rows, int heads, cudaStream_t s) {
    return by_types(dtype, pc.dtype, [&](auto t, auto c) {
        return append_typed<decltype(t), decltype(c)>(pc, qkv, rope, rope_len, row_seq, row_pos, rows, heads, s);
    });
}

// The partials come first, at a size of their own: the tickets of a call never lie where another call's partials were.
size_t attn_paged_ws_bytes(int batch, int heads, int kv_heads) {
    const size_t blocks = static_cast<size_t>((heads / kv_heads - 1) / 8 + 1);
    return kAttnPartBytes + (static_cast<size_t>(batch) * kv_heads * blocks * 4 + 255) / 256 * 256;
}

cudaError_t launch_attn_decode_paged(const PagedCache& pc, int dtype, const void* qkv, const float* rope, int rope_len,
                                     const int* pos, void* out, int heads, void* ws, int num_sms, cudaStream_t s) {
    AttnParams p{};
    p.pc = pc;
    p.qkv = qkv;
    p.rope = reinterpret_cast<const float2*>(rope);
    p.rope_len = rope_len;
    p.pos = pos;
    p.out = out;
    p.heads = heads;
    p.group = heads / pc.kv_heads;
    p.io = dtype;
    p.page_div = FastDiv(static_cast<uint32_t>(pc.page_size));
    p.part = static_cast<float*>(ws);
    p.tickets = reinterpret_cast<int*>(static_cast<char*>(ws) + kAttnPartBytes);
    switch (pc.dtype) {
        case kF32: return attend_typed<float>(p, num_sms, s);
        case kBF16: return attend_typed<__nv_bfloat16>(p, num_sms, s);
        case kF16: return attend_typed<__half>(p, num_sms, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace xl
