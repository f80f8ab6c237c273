// A paged key/value cache: append of rows, and attention of one new token per sequence.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

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
// A copy, bound by its bytes; a CTA takes whole rows (kAppendThreads threads
// over them), so that no index needs a 64-bit division.  16384 rows of 8 heads of
// 128 in bf16: 29 us, 4.9 TB/s; 512 rows of 24 heads of 64 in fp32: 3.8 us.
constexpr int kAppendThreads = 256;
template <typename T, typename C>
__global__ void __launch_bounds__(kAppendThreads) kv_append_paged_kernel(const PagedCache pc, const T* __restrict__ qkv,
                                                                         const float2* __restrict__ rope, int rope_len,
                                                                         const int* __restrict__ row_seq,
                                                                         const int* __restrict__ row_pos, int rows,
                                                                         int heads, int rows_per_cta, FastDiv items_div,
                                                                         FastDiv page_div) {
    const int d = pc.head_dim, per_head = d / 16, per_side = pc.kv_heads * per_head, items = 2 * per_side;
    for (int i = threadIdx.x; i < rows_per_cta * items; i += kAppendThreads) {
        const int in = static_cast<int>(items_div.div(i)), rest = i - in * items;
        const long long r = static_cast<long long>(blockIdx.x) * rows_per_cta + in;
        if (r >= rows) return;
        const int row = static_cast<int>(r);
        const bool value = rest >= per_side;
        const int of = value ? rest - per_side : rest, h = d == 64 ? of >> 2 : of >> 3, part = of & (per_head - 1);
        const int seq = row_seq[row], pos = row_pos[row];
        // the row's elements are on their way while its page is looked up
        const T* src = qkv + static_cast<int64_t>(row) * (heads + 2 * pc.kv_heads) * d +
                       static_cast<int64_t>(heads + (value ? pc.kv_heads : 0) + h) * d;
        const int e0 = value ? part * 16 : part * 8, e1 = value ? e0 + 8 : e0 + d / 2;
        float a[8], b[8];
        load8(src + e0, a);
        load8(src + e1, b);
        if (seq < 0 || seq >= pc.batch || !paged_pos_ok(pos, pc.max_pages, pc.page_size, rope ? rope_len : 0)) continue;
        const int n = static_cast<int>(page_div.div(pos));
        const int page = pc.page_table[static_cast<int64_t>(seq) * pc.max_pages + n];
        if (!paged_valid(page, pc.num_pages)) continue;
        const int64_t at = paged_base(page, h, pc.kv_heads, pc.page_size, d) + static_cast<int64_t>(pos - n * pc.page_size) * d;
        if (!value && rope) {
            const float4* cs = reinterpret_cast<const float4*>(rope + static_cast<int64_t>(pos) * (d / 2) + e0);
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
                const float4 x = cs[k / 2];
                rotate(a[k], b[k], make_float2(x.x, x.y));
                rotate(a[k + 1], b[k + 1], make_float2(x.z, x.w));
            }
        }
        C* dst = static_cast<C*>(value ? pc.v : pc.k) + at;
        store8(dst + e0, a);
        store8(dst + e1, b);
    }
}

// ---- attention of one new token a sequence ------------------------------------------------------------------------
//
//   o = sum_t w_t v_t / sum_t w_t,  w_t = exp(q . k_t / sqrt(d)),  t = 0 .. pos
//
// One pass over the cache with the running maximum and sum of a softmax.  What
// bounds it is reading the cache, so the work is cut by cache bytes: every
// (sequence, key/value head, block of 8 or 16 query heads) is a "pair" of
// chunks of 64 positions, the chunks of all pairs stand in one row, and
// every CTA takes an equal stretch of that row (lengths live on the device; a
// CTA finds its stretch from them).  A pair that one CTA covers is finished
// there; else its CTAs leave (maximum, sum, output) partials in the workspace
// and the last to arrive (a ticket, nobody waits) merges them in CTA order, so
// results do not depend on timing.
//
// Within a CTA each warp takes tiles of 16 positions with its own running
// softmax.  mma.sync does the sums: positions (for the output: columns of the
// values) are its 16 rows, 8 query heads that share the key/value head its
// columns, so a byte of cache is read once for all of them.  The cache goes
// from global memory straight into the MMA's register layout, 16 bytes a
// load: the columns that a lane holds are a permutation of the MMA's, applied
// alike to both operands of the scores (any order of d sums the same) and,
// for the values, undone when the output is stored.  The queries stand in
// shared memory in that layout; the weights change from one MMA's result to
// the next one's operand by an 8 x 8 transpose in registers (movmatrix).
//
// Precision: queries are split in two 16-bit halves, and so are the weights,
// which leaves 2^-17 (bf16) or 2^-23 (fp16) of error where rounding them would
// leave 2^-9 or 2^-12; fp32 rows over a bf16 cache take three parts, which are
// all of an fp32 value; an fp32 cache runs as three TF32 products of split
// operands.  fp16 has no value below 2^-24 and none above 65504: what is split
// for it is scaled by powers of two, the low half by one more, so that a weight
// keeps its 2^-23 down to 2^-29 of the largest (e^-20) and an absolute 2^-52
// below.  Sums, maxima and the running output are fp32.
//
// 64 sequences up to 8192 (32 heads on 8 of 128, bf16): 187 us, 5.8 TB/s; one
// of 131072: 96 us, 5.6 TB/s.  8 sequences up to 768 (24 heads of 64, fp32):
// 16 us, of which reading the cache would be 6.4; the rest is the chain of one
// stretch: finding it 1.6, first loads 2, merging 2.

constexpr int kAttnWarps = 4;
constexpr int kAttnShort = 8;                // chunks a CTA up to which stretches keep to one pair
constexpr int kAttnTries = 6;
constexpr int kMergeAhead = 8;
constexpr int kAttnRows = 16;                // most query heads of a pair
constexpr size_t kAttnSlotFloats = kAttnRows * (128 + 2);
constexpr size_t kAttnPartBytes = kPagedMaxCtas * 2 * kAttnSlotFloats * 4;  // two partials a CTA
constexpr int kTile = 16;                    // positions of a warp's tile
constexpr int kChunk = kAttnWarps * kTile;
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

template <int N, typename T>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    static_assert(N == 2 || N == 4, "2 or 4 elements, aligned to as many");
    if constexpr (sizeof(T) == 4 && N == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else if constexpr (sizeof(T) == 4 || N == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
    } else {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(p);
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
    }
}
template <int N>
__device__ __forceinline__ void load_io_n(const void* p, int64_t i, int io, float (&v)[N]) {
    if (io == kF32) load_n<N>(static_cast<const float*>(p) + i, v);
    else if (io == kBF16) load_n<N>(static_cast<const __nv_bfloat16*>(p) + i, v);
    else load_n<N>(static_cast<const __half*>(p) + i, v);
}
// 16 bytes of shared memory, read where it stands (kept in registers across the tiles they would spill).
__device__ __forceinline__ uint4 load_shared(const uint4* p) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
    return v;
}

__device__ __forceinline__ uint2 load_shared(const uint2* p) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                 : "=r"(v.x), "=r"(v.y)
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
    return v;
}

// fp16 holds 5 exponent bits: a query row is scaled by 2^-row_exponent so that its largest value is in [2^14, 2^15), which
// leaves an element 2^-28 of that its 2^-23.  (A row below 2^-112 is scaled by less; its scores are zeros beside 1.)
template <typename C>
constexpr bool kScaled = false;
template <>
constexpr bool kScaled<__half> = true;
__device__ __forceinline__ int row_exponent(uint32_t bits) {
    const int e = static_cast<int>(bits >> 23) - 127 - 14;
    return bits == 0u || bits >= 0x7f800000u ? 0 : max(-126, e);
}

// What the low half is scaled by: the rounding of the high one is 2^-12 of it at most.
template <typename C>
constexpr float kLowUp = kScaled<C> ? 4096.0f : 1.0f;
// What the weights (at most 1) are scaled by: up to 2^15 is below fp16's largest value.
template <typename C>
constexpr float kWeightUp = kScaled<C> ? 32768.0f : 1.0f;

// What two bf16 halves leave of two values: with it they have 24 bits, fp32's own.
__device__ __forceinline__ uint32_t rest16(float a, float b, uint32_t hi, uint32_t lo) {
    const float2 h = make_float2(__uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u));
    const float2 l = make_float2(__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u));
    return pack_pair((a - h.x) - l.x, (b - h.y) - l.y, __nv_bfloat16{});
}

// Two values as a pair of 16-bit halves: v = hi + lo / kLowUp up to 2^-17 (bf16) or 2^-23 (fp16, from 2^-14 on) of it.
template <typename C>
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const float ha = to_float(from_float<C>(a)), hb = to_float(from_float<C>(b));
    hi = pack_pair(ha, hb, C{});
    lo = pack_pair((a - ha) * kLowUp<C>, (b - hb) * kLowUp<C>, C{});
}
// v = hi + lo for TF32 products: hi to nearest, so that what lo loses (it is
// cut to 11 bits) has no sign of its own.
__device__ __forceinline__ uint32_t tf32_hi(uint32_t v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(__uint_as_float(v)));
    return r;
}
__device__ __forceinline__ uint32_t tf32_lo(uint32_t v, uint32_t hi) {
    return __float_as_uint(__uint_as_float(v) - __uint_as_float(hi));
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
// An 8 x 8 matrix of 16-bit values, lane l holding row l / 4, columns 2 (l % 4) and the next: its transpose, held alike.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_fast(float v) {  // 2^-22 relative, 0 below 2^-126
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// C: cache type, D: head dim, WIDE: 16 query heads a pair (else 8), as two column halves of the MMAs.
// PARTS: 16-bit values that a query or weight is split into.
template <typename C, int D, bool WIDE, int PARTS>
struct AttnShape {
    static constexpr bool k32 = sizeof(C) == 4;
    static constexpr int kVec = 16 / sizeof(C);             // elements of a 16-byte load
    static constexpr int kKch = D / (4 * kVec);             // 16-byte loads of a lane per key row
    static constexpr int kVch = D / (8 * kVec);             // ... per value row
    static constexpr int kSteps = 2 * kKch;                 // MMA steps of a score
    static constexpr int kHalves = WIDE ? 2 : 1;
    static constexpr int kRows = 8 * kHalves;
    static constexpr int kPer = kVec / 2;                   // columns of a lane in a step
    static constexpr int kFragFloats = kSteps * kHalves * (PARTS == 3 ? 192 : 128);
    static constexpr int kPartFloats = kAttnWarps * kRows * (D + 2);
    static constexpr int kSmemFloats = kFragFloats > kPartFloats ? kFragFloats : kPartFloats;
    // CTAs an SM holds, by registers: a lane keeps a tile's keys and values and its part of the output
    // (4 and 5, with spills throughout, took 212 and 306 us where 3 took 194, 64 sequences up to 8192 in bf16).
    // What spills as it is, in bytes stored: an fp32 cache with 9 to 16 heads a pair, 68 at width 128 and 40
    // at 64; 8 or none elsewhere.
    static constexpr int kCtas = D == 128 && (k32 || WIDE) ? 2 : 3;
};

// Where a CTA stands in its stretch and in a pair: kept in shared memory while the tiles run, which need the registers (64
// sequences up to 8192, bf16: 204 us with all of it in registers, of which some were spilled, 187 us so).
struct Stretch {
    long long at, end, first, all, grid, pair_first;
    int b, step, seq, pos, kh, h0, nh, c0, c1, nch, nu, pair;
};

// A warp's tiles of chunks c0 .. c1 again, in plain fp32, where their sums came out as an infinity or NaN.  Split operands
// cannot tell what the definition says of those (0 x inf and inf - inf come up between the halves): here a score of minus
// infinity is a weight of 0, an infinite value under a weight that is not 0 (however small) an infinite output, 0 x inf
// and inf - inf NaN.  (All values infinite, 64 sequences up to 8192: 2.0 ms where finite ones take 0.19.)  2 heads and 4 positions at a time, D / 32 columns a lane; part: the warp's rows of D outputs,
// maximum and sum, as the caller leaves them.
template <typename C, int D>
__device__ __forceinline__ void plain_part(const AttnParams& p, int seq, int kh, int h0, int nh, int pos, int c0, int c1,
                                           bool bad, float* part) {
    constexpr int kCols = D / 32, kHeads = 2, kRow = 4;  // columns lane + 32 i: i and i + kCols / 2 are a rotation's pair
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedCache& pc = p.pc;
    const int* table = pc.page_table + static_cast<int64_t>(seq) * pc.max_pages;
    const C *kp = static_cast<const C*>(pc.k), *vp = static_cast<const C*>(pc.v);
#pragma unroll 1
    for (int r0 = 0; r0 < nh; r0 += kHeads) {  // past the last head: the last one again
        float q[kHeads][kCols], o[kHeads][kCols], past[kHeads][kCols], top[kHeads], sum[kHeads];  // past: infinities, NaN
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const int64_t src = seq * static_cast<int64_t>(p.heads + 2 * pc.kv_heads) * D +
                                static_cast<int64_t>(h0 + min(r0 + h, nh - 1)) * D + lane;
#pragma unroll
            for (int i = 0; i < kCols; ++i) q[h][i] = load_io(p.qkv, src + 32 * i, p.io), o[h][i] = past[h][i] = 0.0f;
            if (p.rope) {
#pragma unroll
                for (int i = 0; i < kCols / 2; ++i)
                    rotate(q[h][i], q[h][i + kCols / 2], p.rope[static_cast<int64_t>(pos) * (D / 2) + lane + 32 * i]);
            }
            top[h] = -INFINITY, sum[h] = 0.0f;
        }
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
#pragma unroll 1
            for (int t = 0; t < kTile; t += kRow) {
                const int x0 = c * kChunk + warp * kTile + t;
                if (x0 > pos) break;
                float k[kRow][kCols], v[kRow][kCols];
#pragma unroll
                for (int u = 0; u < kRow; ++u) {
                    const int x = min(x0 + u, pos), n = static_cast<int>(p.page_div.div(x)), page = table[n];
                    const int64_t at = paged_base(paged_valid(page, pc.num_pages) ? page : 0, kh, pc.kv_heads, pc.page_size, D) +
                                       static_cast<int64_t>(x - n * pc.page_size) * D + lane;
#pragma unroll
                    for (int i = 0; i < kCols; ++i) k[u][i] = to_float(__ldcg(kp + at + 32 * i)), v[u][i] = to_float(__ldcg(vp + at + 32 * i));
                }
#pragma unroll
                for (int u = 0; u < kRow; ++u) {
                    if (x0 + u > pos) break;
                    float s[kHeads];
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        s[h] = 0.0f;
#pragma unroll
                        for (int i = 0; i < kCols; ++i) s[h] = fmaf(q[h][i], k[u][i], s[h]);
                    }
#pragma unroll
                    for (int h = 0; h < kHeads; ++h) {
                        s[h] = warp_sum(s[h]) * (kLog2e / (D == 64 ? 8.0f : 11.313708498984761f));
                        const bool out = s[h] == -INFINITY;
                        const float high = fmaxf(top[h], s[h]), old = top[h] == -INFINITY ? 0.0f : exp2_fast(top[h] - high);
                        const float w = out ? 0.0f : exp2_fast(s[h] - high);
                        top[h] = high, sum[h] = sum[h] * old + w;
#pragma unroll
                        for (int i = 0; i < kCols; ++i) {
                            const bool finite = fabsf(v[u][i]) < INFINITY;
                            o[h][i] = o[h][i] * old + (finite ? w * v[u][i] : 0.0f);
                            if (!finite) past[h][i] += out ? __int_as_float(0x7fffffff) : v[u][i];
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            float* row = part + min(r0 + h, nh - 1) * (D + 2);
#pragma unroll
            for (int i = 0; i < kCols; ++i) row[lane + 32 * i] = o[h][i] + past[h][i];
            if (lane == 0) row[D] = top[h], row[D + 1] = bad ? __int_as_float(0x7fffffff) : sum[h];
        }
    }
}

// A partial output under its factor; an infinite one stays so where the factor is below the floats' range.
__device__ __forceinline__ float under(float f, float o) { return fabsf(o) == INFINITY ? o : f * o; }

template <typename C, int D, bool WIDE, int PARTS>
__global__ void __launch_bounds__(128, (AttnShape<C, D, WIDE, PARTS>::kCtas))
    attn_decode_paged_kernel(const __grid_constant__ AttnParams p) {
    using S = AttnShape<C, D, WIDE, PARTS>;
    extern __shared__ __align__(16) float smem[];
    uint4* frag = reinterpret_cast<uint4*>(smem);  // [steps][halves][32]: the queries in the MMA's layout, hi and lo
    uint2* frag3 = reinterpret_cast<uint2*>(frag + S::kSteps * S::kHalves * 32);  // their third parts, where there are such
    float* warp_part = smem;                       // [warps][rows][D + 2], once the queries are no longer read
    __shared__ int flag;
    __shared__ uint32_t row_max[16];
    __shared__ Stretch held_back;
    const PagedCache& pc = p.pc;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pairs = pc.kv_heads * p.blocks;  // of a sequence
    const int64_t width = static_cast<int64_t>(p.heads + 2 * pc.kv_heads) * D;
    C *kp = static_cast<C*>(pc.k), *vp = static_cast<C*>(pc.v);
    const int limit = p.rope ? p.rope_len : 0;

    auto chunks_of = [&](int pos) {
        return paged_pos_ok(pos, pc.max_pages, pc.page_size, limit) ? pos / kChunk + 1 : 1;
    };
    // The stretches are counted in units of `step` chunks of a pair.  Every warp adds up all sequences' units and
    // finds the sequence that its CTA's stretch begins in; the positions are read once where a warp holds them all.
    const int held = lane < pc.batch ? chunks_of(p.pos[lane]) : 0;
    auto chunks_at = [&](int i) { return i < 32 ? held : i < pc.batch ? chunks_of(p.pos[i]) : 0; };
    auto units_in_all = [&](unsigned step) {
        long long total = 0;  // a sequence has at most 2^25 chunks, 32 of them fit 32 bits
        for (int b0 = 0; b0 < pc.batch; b0 += 32)
            total += __reduce_add_sync(0xffffffffu, static_cast<unsigned>(chunks_at(b0 + lane) + step - 1) / step);
        return total * pairs;
    };
    // Short work: the step is raised until every CTA has one unit at most, so that none takes parts of two pairs one
    // after the other.  Long work, and more pairs than CTAs: single chunks, which cuts evenly.
    int step = 1;
    long long all = units_in_all(1);
    if (all > gridDim.x && all <= static_cast<long long>(gridDim.x) * kAttnShort) {
        int least = static_cast<int>((all + gridDim.x - 1) / gridDim.x);
        for (int tries = 0; tries < kAttnTries; ++tries, ++least) {
            const long long units = units_in_all(least);
            if (units <= gridDim.x) {
                step = least, all = units;
                break;
            }
        }
    }
    long long grid = min(static_cast<long long>(gridDim.x), all);  // a unit at least for every CTA that works
    if (blockIdx.x >= grid) return;
    bool brief = paged_brief(all);
    long long at = paged_share(blockIdx.x, all, grid, brief);
    long long end = paged_share(blockIdx.x + 1, all, grid, brief);
    int b = 0;
    long long first = 0;  // the row's index of sequence b's first unit
    for (int b0 = 0; b0 < pc.batch; b0 += 32) {
        const unsigned own = static_cast<unsigned>(chunks_at(b0 + lane) + step - 1) / static_cast<unsigned>(step);
        unsigned upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, first + static_cast<long long>(upto) * pairs > at);
        if (past) {
            const int i = __ffs(past) - 1;
            b = b0 + i;
            first += static_cast<long long>(__shfl_sync(0xffffffffu, upto - own, i)) * pairs;
            break;
        }
        first += static_cast<long long>(__shfl_sync(0xffffffffu, upto, 31)) * pairs;
    }

    while (at < end) {
        const int pos = p.pos[b];
        const int nch = chunks_of(pos), nu = (nch + step - 1) / step;
        const int pair = brief ? static_cast<int>(at - first) / nu : static_cast<int>((at - first) / nu);
        const int u0 = static_cast<int>((at - first) - static_cast<long long>(pair) * nu);
        const int u1 = static_cast<int>(min(static_cast<long long>(nu), u0 + (end - at)));
        const int c0 = u0 * step, c1 = min(nch, u1 * step);
        const int kh = pair / p.blocks, blk = pair - kh * p.blocks;
        const int h0 = kh * p.group + blk * S::kRows, nh = min(S::kRows, p.group - blk * S::kRows);
        const long long pair_first = first + static_cast<long long>(pair) * nu;
        const int seq = b;
        at += u1 - u0;
        if (pair == pairs - 1 && u1 == nu) {
            first += static_cast<long long>(pairs) * nu;
            ++b;
        }
        if (!paged_pos_ok(pos, pc.max_pages, pc.page_size, limit)) {
            const float v = pos == -1 ? 0.0f : __int_as_float(0x7fffffff);
            const int64_t out0 = (static_cast<int64_t>(seq) * p.heads + h0) * D;
            for (int i = threadIdx.x; i < nh * D; i += 128) store_io(p.out, out0 + i, v, p.io);
            continue;
        }
        const int* table = pc.page_table + static_cast<int64_t>(seq) * pc.max_pages;
        const int64_t qrow = seq * width;

        __syncthreads();  // the last pair's shared memory has been read

        // Rows of the pool that a tile's positions are in, a position a lane.  Positions past the last one stand for
        // the last one: their scores are masked, and no lane reads what no position holds.
        bool bad = false;
        auto find_rows = [&](int c) {
            const int x = min(c * kChunk + warp * kTile + (lane & (kTile - 1)), pos);
            const int n = static_cast<int>(p.page_div.div(x));
            int page = table[n];
            if (!paged_valid(page, pc.num_pages)) {
                bad = true;
                page = 0;
            }
            return static_cast<uint32_t>((static_cast<int64_t>(page) * pc.kv_heads + kh) * pc.page_size + (x - n * pc.page_size));
        };
        uint4 kr[2][S::kKch], vr[4][S::kVch];  // key rows g and g + 8; value rows 2t, 2t + 1, 2t + 8, 2t + 9
        auto load_k = [&](uint32_t rows) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t r = __shfl_sync(0xffffffffu, rows, 8 * n + g);
                const uint4* src = reinterpret_cast<const uint4*>(kp + static_cast<int64_t>(r) * D) + t;
#pragma unroll
                for (int j = 0; j < S::kKch; ++j) kr[n][j] = __ldcg(src + 4 * j);
            }
        };
        auto load_v = [&](uint32_t rows) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t r = __shfl_sync(0xffffffffu, rows, 8 * (n >> 1) + 2 * t + (n & 1));
                const uint4* src = reinterpret_cast<const uint4*>(vp + static_cast<int64_t>(r) * D) + g;
#pragma unroll
                for (int j = 0; j < S::kVch; ++j) vr[n][j] = __ldcg(src + 8 * j);
            }
        };
        // The first tile is on its way before the queries are made, unless it holds the position to be written here.
        const uint32_t rows = find_rows(c0);
        const bool early = c0 * kChunk + (warp + 1) * kTile <= pos;
        if (early) {
            load_k(rows);
            load_v(rows);
        }

        // The CTA that holds the last position writes its key and value (read here, written when the queries are made).
        int64_t new_at = -1;
        float new_row[4];
        float2 new_cs = make_float2(1.0f, 0.0f);
        if (c1 == nch && threadIdx.x < D / 2) {
            const int n = static_cast<int>(p.page_div.div(pos)), page = table[n], j = threadIdx.x;
            const int64_t src = qrow + static_cast<int64_t>(p.heads + kh) * D + j, sv = src + static_cast<int64_t>(pc.kv_heads) * D;
            new_row[0] = load_io(p.qkv, src, p.io), new_row[1] = load_io(p.qkv, src + D / 2, p.io);
            new_row[2] = load_io(p.qkv, sv, p.io), new_row[3] = load_io(p.qkv, sv + D / 2, p.io);
            if (p.rope) new_cs = p.rope[static_cast<int64_t>(pos) * (D / 2) + j];
            if (paged_valid(page, pc.num_pages))
                new_at = paged_base(page, kh, pc.kv_heads, pc.page_size, D) + static_cast<int64_t>(pos - n * pc.page_size) * D + j;
        }

        // The rotated queries, each lane's columns of each step, split in hi and lo.  Columns j and j + d/2 are half
        // the steps apart, so a thread rotates and writes two steps.
        if constexpr (kScaled<C>) {
            if (threadIdx.x < 16) row_max[threadIdx.x] = 0u;
            __syncthreads();
        }
        constexpr int kItems = S::kHalves * (S::kSteps / 2) * 32;
        constexpr int kEach = (kItems + 127) / 128;
        float qa[kEach][S::kPer], qb[kEach][S::kPer];
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = threadIdx.x + 128 * n, l = i & 31, st = (i >> 5) % (S::kSteps / 2), half = (i >> 5) / (S::kSteps / 2);
            const int r = (l >> 2) + 8 * half, e0 = (4 * (st / 2) + (l & 3)) * S::kVec + (st & 1) * S::kPer;
#pragma unroll
            for (int k = 0; k < S::kPer; ++k) qa[n][k] = qb[n][k] = 0.0f;
            if (i < kItems && r < nh) {
                const int64_t src = qrow + static_cast<int64_t>(h0 + r) * D + e0;
                load_io_n<S::kPer>(p.qkv, src, p.io, qa[n]);
                load_io_n<S::kPer>(p.qkv, src + D / 2, p.io, qb[n]);
                if (p.rope) {
                    const float4* cs = reinterpret_cast<const float4*>(p.rope + static_cast<int64_t>(pos) * (D / 2) + e0);
#pragma unroll
                    for (int k = 0; k < S::kPer; k += 2) {
                        const float4 x = cs[k / 2];
                        rotate(qa[n][k], qb[n][k], make_float2(x.x, x.y));
                        rotate(qa[n][k + 1], qb[n][k + 1], make_float2(x.z, x.w));
                    }
                }
                if constexpr (kScaled<C>) {
                    float big = 0.0f;
#pragma unroll
                    for (int k = 0; k < S::kPer; ++k) big = fmaxf(big, fmaxf(fabsf(qa[n][k]), fabsf(qb[n][k])));
                    atomicMax(&row_max[r], __float_as_uint(big));
                }
            }
        }
        if constexpr (kScaled<C>) __syncthreads();
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = threadIdx.x + 128 * n, l = i & 31, st = (i >> 5) % (S::kSteps / 2), half = (i >> 5) / (S::kSteps / 2);
            if (i >= kItems) break;
            float down = 1.0f;
            if constexpr (kScaled<C>) down = __uint_as_float(static_cast<uint32_t>(127 - row_exponent(row_max[(l >> 2) + 8 * half])) << 23);
            uint4 *fa = frag + (st * S::kHalves + half) * 32 + l, *fb = fa + (S::kSteps / 2) * S::kHalves * 32;
            if constexpr (S::k32) {
                const uint32_t a0 = __float_as_uint(qa[n][0]), a1 = __float_as_uint(qa[n][1]);
                const uint32_t b0 = __float_as_uint(qb[n][0]), b1 = __float_as_uint(qb[n][1]);
                const uint32_t ha0 = tf32_hi(a0), ha1 = tf32_hi(a1), hb0 = tf32_hi(b0), hb1 = tf32_hi(b1);
                *fa = make_uint4(ha0, ha1, tf32_lo(a0, ha0), tf32_lo(a1, ha1));
                *fb = make_uint4(hb0, hb1, tf32_lo(b0, hb0), tf32_lo(b1, hb1));
            } else {
                uint4 o;
                split16<C>(qa[n][0] * down, qa[n][1] * down, o.x, o.z);
                split16<C>(qa[n][S::kPer - 2] * down, qa[n][S::kPer - 1] * down, o.y, o.w);
                *fa = o;
                if constexpr (PARTS == 3)
                    frag3[fa - frag] = make_uint2(rest16(qa[n][0], qa[n][1], o.x, o.z),
                                                  rest16(qa[n][S::kPer - 2], qa[n][S::kPer - 1], o.y, o.w));
                split16<C>(qb[n][0] * down, qb[n][1] * down, o.x, o.z);
                split16<C>(qb[n][S::kPer - 2] * down, qb[n][S::kPer - 1] * down, o.y, o.w);
                *fb = o;
                if constexpr (PARTS == 3)
                    frag3[fb - frag] = make_uint2(rest16(qb[n][0], qb[n][1], o.x, o.z),
                                                  rest16(qb[n][S::kPer - 2], qb[n][S::kPer - 1], o.y, o.w));
            }
        }
        if (new_at >= 0) {
            if (p.rope) rotate(new_row[0], new_row[1], new_cs);
            kp[new_at] = from_float<C>(new_row[0]), kp[new_at + D / 2] = from_float<C>(new_row[1]);
            vp[new_at] = from_float<C>(new_row[2]), vp[new_at + D / 2] = from_float<C>(new_row[3]);
        }
        if (threadIdx.x == 0)
            held_back = Stretch{at, end, first, all, grid, pair_first, b, step, seq, pos, kh, h0, nh, c0, c1, nch, nu, pair};
        __syncthreads();  // queries, and the new rows, are there for every warp
        if (!early) {
            load_k(rows);
            load_v(rows);
        }
        // turn a head's products into log2 of its weights (heads 2t and 2t + 1 of each half)
        float back[S::kHalves][2];
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                back[h][j] = kLog2e / (D == 64 ? 8.0f : 11.313708498984761f);
                if constexpr (kScaled<C>)
                    back[h][j] *= __uint_as_float(static_cast<uint32_t>(127 + row_exponent(row_max[8 * h + 2 * t + j])) << 23);
            }

        float top[S::kHalves][2], sum[S::kHalves][2], acc[S::kHalves][D / 16][4];
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h) {
            top[h][0] = top[h][1] = -INFINITY, sum[h][0] = sum[h][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[h][i][j] = 0.0f;
        }
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
            const int x0 = c * kChunk + warp * kTile;
            if (x0 > pos) break;  // only the last chunk has tiles past the end
            const uint32_t next = find_rows(c + 1);
            // The MMA cuts its sums instead of rounding them, so long sums are kept out of it: the 8 or 16 large products
            // of an fp32 cache in two halves, added here; the outputs tile by tile.
            float s[S::kHalves][4], also[S::kHalves][4], more[S::kHalves][4];
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[h][j] = also[h][j] = more[h][j] = 0.0f;
#pragma unroll
            for (int i = 0; i < S::kSteps; ++i) {
                const int w = (i & 1) * 2;
                const uint32_t a[4] = {word(kr[0][i / 2], w), word(kr[1][i / 2], w), word(kr[0][i / 2], w + 1), word(kr[1][i / 2], w + 1)};
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h) {
                    const uint4 q = load_shared(frag + (i * S::kHalves + h) * 32 + lane);
                    float(&large)[4] = S::k32 && (i & 1) ? also[h] : s[h];
                    if constexpr (S::k32) {
                        const uint32_t hi[4] = {tf32_hi(a[0]), tf32_hi(a[1]), tf32_hi(a[2]), tf32_hi(a[3])};
                        const uint32_t lo[4] = {tf32_lo(a[0], hi[0]), tf32_lo(a[1], hi[1]), tf32_lo(a[2], hi[2]),
                                                tf32_lo(a[3], hi[3])};
                        mma_tf32(large, hi, q.x, q.y);
                        mma_tf32(more[h], hi, q.z, q.w);
                        mma_tf32(more[h], lo, q.x, q.y);
                    } else {
                        mma16(large, a, q.x, q.y, C{});
                        if constexpr (PARTS == 3) {
                            const uint2 q3 = load_shared(frag3 + (i * S::kHalves + h) * 32 + lane);
                            mma16(more[h], a, q3.x, q3.y, C{});
                        }
                        mma16(more[h], a, q.z, q.w, C{});
                    }
                }
            }
            load_k(next);
            float old[S::kHalves][2];
            bool raise = false;
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[h][j] = (s[h][j] + also[h][j] + more[h][j] * (1.0f / kLowUp<C>)) * back[h][j & 1];
                if (x0 + kTile > pos + 1) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (x0 + g + (j >> 1) * 8 > pos) s[h][j] = -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float high = fmaxf(s[h][j], s[h][j + 2]);
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 4));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 8));
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 16));
                    high = fmaxf(high, top[h][j]);
                    old[h][j] = exp2_fast(top[h][j] - high);
                    raise |= high != top[h][j];
                    top[h][j] = high;
                    s[h][j] = exp2_fast(s[h][j] - high);
                    s[h][j + 2] = exp2_fast(s[h][j + 2] - high);
                    sum[h][j] = sum[h][j] * old[h][j] + (s[h][j] + s[h][j + 2]);
                }
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[h][i][j] *= old[h][j & 1];
            }
            // The weights as the next MMAs' second operand: head g, positions 2t, 2t + 1 and those + 8.
            uint32_t wh[S::kHalves][4], wl[S::kHalves][4], w3[S::kHalves][2];
#pragma unroll
            for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if constexpr (S::k32) {
                        const uint32_t x = __float_as_uint(s[h][2 * n]), y = __float_as_uint(s[h][2 * n + 1]);
                        const uint32_t up = transpose8(__byte_perm(x, y, 0x7632)), down = transpose8(__byte_perm(x, y, 0x5410));
                        const uint32_t w0 = __byte_perm(down, up, 0x5410), w1 = __byte_perm(down, up, 0x7632);
                        wh[h][2 * n] = tf32_hi(w0), wh[h][2 * n + 1] = tf32_hi(w1);
                        wl[h][2 * n] = tf32_lo(w0, wh[h][2 * n]), wl[h][2 * n + 1] = tf32_lo(w1, wh[h][2 * n + 1]);
                    } else {
                        uint32_t hi, lo;
                        split16<C>(s[h][2 * n] * kWeightUp<C>, s[h][2 * n + 1] * kWeightUp<C>, hi, lo);
                        wh[h][n] = transpose8(hi), wl[h][n] = transpose8(lo);
                        if constexpr (PARTS == 3) w3[h][n] = transpose8(rest16(s[h][2 * n], s[h][2 * n + 1], hi, lo));
                    }
                }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const int ch = i / (S::kVec / 2), e = i % (S::kVec / 2);
                float o[S::kHalves][4], low[S::kHalves][4];  // low: of the low halves, where they are scaled
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[h][j] = low[h][j] = 0.0f;
                if constexpr (S::k32) {
                    // position 2t is the MMA's k = t, 2t + 1 its k = t + 4; columns 2e and 2e + 1 its rows g and g + 8
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const uint32_t a[4] = {word(vr[2 * n][ch], 2 * e), word(vr[2 * n][ch], 2 * e + 1),
                                               word(vr[2 * n + 1][ch], 2 * e), word(vr[2 * n + 1][ch], 2 * e + 1)};
                        const uint32_t hi[4] = {tf32_hi(a[0]), tf32_hi(a[1]), tf32_hi(a[2]), tf32_hi(a[3])};
                        const uint32_t lo[4] = {tf32_lo(a[0], hi[0]), tf32_lo(a[1], hi[1]), tf32_lo(a[2], hi[2]),
                                                tf32_lo(a[3], hi[3])};
#pragma unroll
                        for (int h = 0; h < S::kHalves; ++h) {
                            mma_tf32(o[h], lo, wh[h][2 * n], wh[h][2 * n + 1]);
                            mma_tf32(o[h], hi, wl[h][2 * n], wl[h][2 * n + 1]);
                            mma_tf32(o[h], hi, wh[h][2 * n], wh[h][2 * n + 1]);
                        }
                    }
                } else {
                    const uint32_t x = word(vr[0][ch], e), y = word(vr[1][ch], e), z = word(vr[2][ch], e), u = word(vr[3][ch], e);
                    const uint32_t a[4] = {__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632), __byte_perm(z, u, 0x5410),
                                           __byte_perm(z, u, 0x7632)};
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h) {
                        if constexpr (PARTS == 3) mma16(o[h], a, w3[h][0], w3[h][1], C{});
                        mma16(kScaled<C> ? low[h] : o[h], a, wl[h][0], wl[h][1], C{});
                        mma16(o[h], a, wh[h][0], wh[h][1], C{});
                    }
                }
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[h][i][j] += kScaled<C> ? o[h][j] + low[h][j] * (1.0f / kLowUp<C>) : o[h][j];
            }
            load_v(next);
        }

        __syncthreads();  // the queries have been read
        const Stretch now = held_back;
        at = now.at, end = now.end, first = now.first, all = now.all, grid = now.grid, b = now.b, step = now.step;
        brief = paged_brief(all);
        const int64_t out0 = (static_cast<int64_t>(now.seq) * p.heads + now.h0) * D;
        // The warps' rows: output parts, then maximum and sum.
        bad = __any_sync(0xffffffffu, bad);
        float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN where a sum is not finite
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                odd[j] = fmaf(sum[h][j & 1], 0.0f, odd[j]);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) odd[j] = fmaf(acc[h][i][j], 0.0f, odd[j]);
            }
        const bool again = __any_sync(0xffffffffu, (odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.0f);
        if (again) plain_part<C, D>(p, now.seq, now.kh, now.h0, now.nh, now.pos, now.c0, now.c1, bad, warp_part + warp * S::kRows * (D + 2));
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (again) break;
                float l = sum[h][j];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
                if (bad) l = __int_as_float(0x7fffffff);
                float* row = warp_part + (warp * S::kRows + 8 * h + 2 * t + j) * (D + 2);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const int d = (i / (S::kVec / 2)) * 8 * S::kVec + S::kVec * g + 2 * (i % (S::kVec / 2));
                    row[d] = acc[h][i][j] * (1.0f / kWeightUp<C>);
                    row[d + 1] = acc[h][i][j + 2] * (1.0f / kWeightUp<C>);
                }
                if (g == 0) row[D] = top[h][j], row[D + 1] = l;
            }
        __syncthreads();
        const bool whole = now.c0 == 0 && now.c1 == now.nch;
        const int slot = 2 * blockIdx.x + (now.c0 > 0 ? 0 : 1);
        float* mine = p.part + slot * static_cast<int64_t>(S::kRows * (D + 2));
        for (int i = threadIdx.x; i < now.nh * D; i += 128) {
            const int r = i / D, d = i - r * D;
            const float* row = warp_part + r * (D + 2);
            float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, row[w * S::kRows * (D + 2) + D]);
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float* x = row + w * S::kRows * (D + 2);
                const float f = x[D] == -INFINITY ? 0.0f : exp2f(x[D] - m);
                l += f * x[D + 1], o += under(f, x[d]);
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
        const int cta0 = paged_owner(now.pair_first, all, grid, brief), cta1 = paged_owner(now.pair_first + now.nu - 1, all, grid, brief);
        int* ticket = p.tickets + static_cast<int64_t>(now.seq) * pairs + now.pair;
        __syncthreads();  // the partial is written; one thread's fence carries it to the others' reads
        if (threadIdx.x == 0) {
            __threadfence();
            flag = atomicAdd(ticket, 1) == cta1 - cta0;
            __threadfence();
        }
        __syncthreads();
        if (!flag) continue;
        // A warp a head, 4 columns a lane (d = 64: half a warp takes every other partial), kMergeAhead partials in
        // flight: a long sequence alone has dozens of them, and one at a time would cost a memory round trip each.
        constexpr int kLanes = D / 4, kApart = 32 / kLanes;
        for (int r = warp; r < now.nh; r += kAttnWarps) {
            float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int d = (lane % kLanes) * 4;
            for (int c = cta0; c <= cta1; c += kMergeAhead * kApart) {
                float2 ml[kMergeAhead];
                float2 x[kMergeAhead][2];
#pragma unroll
                for (int k = 0; k < kMergeAhead; ++k) {
                    const int from = c + k * kApart + lane / kLanes;
                    // a pair's first CTA leaves it in the second slot: its stretch ends with the pair's beginning
                    const float* src = p.part + (2 * min(from, cta1) + (min(from, cta1) == cta0 ? 1 : 0)) *
                                                    static_cast<int64_t>(S::kRows * (D + 2)) + r * (D + 2);
                    ml[k] = __ldcg(reinterpret_cast<const float2*>(src + D));
                    x[k][0] = __ldcg(reinterpret_cast<const float2*>(src + d));
                    x[k][1] = __ldcg(reinterpret_cast<const float2*>(src + d + 2));
                    if (from > cta1) ml[k] = make_float2(-INFINITY, 0.0f);
                }
#pragma unroll
                for (int k = 0; k < kMergeAhead; ++k) {
                    const float up = fmaxf(m, ml[k].x);
                    const float f0 = m == -INFINITY ? 0.0f : exp2_fast(m - up);
                    const float f1 = ml[k].x == -INFINITY ? 0.0f : exp2_fast(ml[k].x - up);
                    l = ml[k].y != ml[k].y ? ml[k].y : l * f0 + ml[k].y * f1;
                    o[0] = under(f0, o[0]) + under(f1, x[k][0].x), o[1] = under(f0, o[1]) + under(f1, x[k][0].y);
                    o[2] = under(f0, o[2]) + under(f1, x[k][1].x), o[3] = under(f0, o[3]) + under(f1, x[k][1].y);
                    m = up;
                }
            }
            if (kApart == 2) {
                const float m2 = __shfl_xor_sync(0xffffffffu, m, 16), l2 = __shfl_xor_sync(0xffffffffu, l, 16);
                const float up = fmaxf(m, m2);
                const float f0 = m == -INFINITY ? 0.0f : exp2_fast(m - up), f1 = m2 == -INFINITY ? 0.0f : exp2_fast(m2 - up);
                l = l != l || l2 != l2 ? __int_as_float(0x7fffffff) : l * f0 + l2 * f1;
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = under(f0, o[k]) + under(f1, __shfl_xor_sync(0xffffffffu, o[k], 16));
            }
            if (lane < kLanes) {
#pragma unroll
                for (int k = 0; k < 4; ++k) store_io(p.out, out0 + r * D + d + k, o[k] / l, p.io);
            }
        }
        if (threadIdx.x == 0) *ticket = 0;
    }
}

template <typename T, typename C>
cudaError_t append_typed(const PagedCache& pc, const void* qkv, const float* rope, int rope_len, const int* row_seq,
                         const int* row_pos, int rows, int heads, cudaStream_t s) {
    const long long items = static_cast<long long>(pc.kv_heads) * (pc.head_dim / 8);
    if (items > 0x3fffffff) return cudaErrorInvalidValue;
    const int each = static_cast<int>(items), per_cta = std::max(1, kAppendThreads / each);
    count_launch();
    kv_append_paged_kernel<T, C><<<(rows - 1) / per_cta + 1, kAppendThreads, 0, s>>>(
        pc, static_cast<const T*>(qkv), reinterpret_cast<const float2*>(rope), rope_len, row_seq, row_pos, rows, heads,
        per_cta, FastDiv(static_cast<uint32_t>(each)), FastDiv(static_cast<uint32_t>(pc.page_size)));
    return cudaGetLastError();
}

template <typename C, int D, bool WIDE, int PARTS = 2>
cudaError_t attend_shape(AttnParams p, int num_sms, cudaStream_t s) {
    // fp32 rows over a bf16 cache take a third part: 64 sequences up to 8192, 32 heads on 8: 194 us and 2.5e-7 of the output
    // off, where two parts take 181 and leave 3.2e-6. The rounding of 16-bit rows (1.7e-3) hides that: 186 us against 192.
    if constexpr (std::is_same_v<C, __nv_bfloat16> && PARTS == 2)
        if (p.io == kF32) return attend_shape<C, D, WIDE, 3>(p, num_sms, s);
    using S = AttnShape<C, D, WIDE, PARTS>;
    p.blocks = (p.group - 1) / S::kRows + 1;
    const long long longest = static_cast<long long>(p.pc.max_pages) * p.pc.page_size;
    const long long chunks = ((longest - 1) / kChunk + 1) * p.pc.batch * p.pc.kv_heads * p.blocks;
    const long long most = std::min(num_sms * S::kCtas, kPagedMaxCtas);
    count_launch();
    attn_decode_paged_kernel<C, D, WIDE, PARTS>
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
