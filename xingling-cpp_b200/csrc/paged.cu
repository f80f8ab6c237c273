// A paged key/value cache: append of rows, and attention of one new token per sequence.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

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

// The new token's key and value, then one warp per (sequence, head): d / 32 elements a lane, one position at a time.
template <typename T, typename C, int D>
__global__ void __launch_bounds__(32) attn_decode_paged_kernel(const PagedCache pc, const T* __restrict__ qkv,
                                                               const float2* __restrict__ rope, int rope_len,
                                                               const int* __restrict__ posv, T* __restrict__ out,
                                                               int heads) {
    constexpr int P = D / 64;  // pairs a lane
    const int b = blockIdx.x / heads, h = blockIdx.x % heads, lane = threadIdx.x;
    const int group = heads / pc.kv_heads, kh = h / group;
    const int pos = posv[b];
    T* o = out + (static_cast<int64_t>(b) * heads + h) * D;
    const bool ok = paged_pos_ok(pos, pc.max_pages, pc.page_size, rope ? rope_len : 0);
    if (!ok) {
        for (int e = lane; e < D; e += 32) o[e] = from_float<T>(pos == -1 ? 0.0f : __int_as_float(0x7fffffff));
        return;
    }
    const T* row = qkv + static_cast<int64_t>(b) * (heads + 2 * pc.kv_heads) * D;
    const int* table = pc.page_table + static_cast<int64_t>(b) * pc.max_pages;
    C *kp = static_cast<C*>(pc.k), *vp = static_cast<C*>(pc.v);
    float q[2 * P], kn[2 * P], vn[2 * P], acc[2 * P];
    bool bad = false;
    const int page = table[pos / pc.page_size];
    const int64_t at = paged_valid(page, pc.num_pages)
                           ? paged_base(page, kh, pc.kv_heads, pc.page_size, D) + static_cast<int64_t>(pos % pc.page_size) * D
                           : -1;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int j = lane + 32 * i;
        float2 cs = make_float2(1.0f, 0.0f);
        if (rope) cs = rope[static_cast<int64_t>(pos) * (D / 2) + j];
        q[2 * i] = to_float(row[h * D + j]), q[2 * i + 1] = to_float(row[h * D + j + D / 2]);
        const T* kr = row + static_cast<int64_t>(heads + kh) * D;
        const T* vr = kr + static_cast<int64_t>(pc.kv_heads) * D;
        kn[2 * i] = to_float(kr[j]), kn[2 * i + 1] = to_float(kr[j + D / 2]);
        if (rope) {
            rotate(q[2 * i], q[2 * i + 1], cs);
            rotate(kn[2 * i], kn[2 * i + 1], cs);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int e = j + t * (D / 2);
            const C kc = from_float<C>(kn[2 * i + t]), vc = from_float<C>(to_float(vr[e]));
            if (at >= 0 && h % group == 0) kp[at + e] = kc, vp[at + e] = vc;
            kn[2 * i + t] = to_float(kc), vn[2 * i + t] = to_float(vc);
            acc[2 * i + t] = 0.0f;
        }
    }
    float top = -INFINITY, sum = 0.0f;
    const float scale = 1.0f / sqrtf(static_cast<float>(D));
    for (int t = 0; t <= pos; ++t) {
        const int pg = table[t / pc.page_size];
        if (!paged_valid(pg, pc.num_pages)) {
            bad = true;
            break;
        }
        const int64_t src = paged_base(pg, kh, pc.kv_heads, pc.page_size, D) + static_cast<int64_t>(t % pc.page_size) * D;
        float s = 0.0f, v[2 * P];
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) {
            const int e = lane + 32 * (i / 2) + (i & 1) * (D / 2);
            s = fmaf(q[i], t == pos ? kn[i] : to_float(kp[src + e]), s);
            v[i] = t == pos ? vn[i] : to_float(vp[src + e]);
        }
        s = warp_sum(s) * scale;
        const float next = fmaxf(top, s), w = expf(s - next), old = expf(top - next);
        sum = sum * old + w;
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) acc[i] = acc[i] * old + w * v[i];
        top = next;
    }
#pragma unroll
    for (int i = 0; i < 2 * P; ++i)
        o[lane + 32 * (i / 2) + (i & 1) * (D / 2)] = from_float<T>(bad ? __int_as_float(0x7fffffff) : acc[i] / sum);
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

template <typename T, typename C>
cudaError_t attend_typed(const PagedCache& pc, const void* qkv, const float* rope, int rope_len, const int* pos, void* out,
                         int heads, cudaStream_t s) {
    const float2* r2 = reinterpret_cast<const float2*>(rope);
    count_launch();
    const int grid = pc.batch * heads;
    if (pc.head_dim == 64)
        attn_decode_paged_kernel<T, C, 64><<<grid, 32, 0, s>>>(pc, static_cast<const T*>(qkv), r2, rope_len, pos,
                                                               static_cast<T*>(out), heads);
    else
        attn_decode_paged_kernel<T, C, 128><<<grid, 32, 0, s>>>(pc, static_cast<const T*>(qkv), r2, rope_len, pos,
                                                                static_cast<T*>(out), heads);
    return cudaGetLastError();
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

size_t attn_paged_ws_bytes(int, int, int) { return 256; }

cudaError_t launch_attn_decode_paged(const PagedCache& pc, int dtype, const void* qkv, const float* rope, int rope_len,
                                     const int* pos, void* out, int heads, void*, int, cudaStream_t s) {
    return by_types(dtype, pc.dtype, [&](auto t, auto c) {
        return attend_typed<decltype(t), decltype(c)>(pc, qkv, rope, rope_len, pos, out, heads, s);
    });
}

}  // namespace xl
