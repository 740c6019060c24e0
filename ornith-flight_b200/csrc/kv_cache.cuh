// kv_cache.cuh — what the attention-cache operators share: the argument checks
// of ofb_kv_cache, element types, and the way from (sequence, entry) to a page.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ofb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements (16-byte aligned address), as f32.
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = to_f32(e[i]);
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    uint4 u;
    T *e = reinterpret_cast<T *>(&u);
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4 *>(p) = u;
}

// Division of entry numbers (below 2^31) by a launch constant: one high product
// and a shift instead of the ~30 instructions of a division.
struct FastDiv {
    uint32_t d, mul, shift;
    __device__ __forceinline__ int div(int n) const {
        return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift);
    }
};
inline FastDiv fast_div(int d) {
    FastDiv f;
    f.d = (uint32_t)d;
    f.shift = 0;
    while ((1u << f.shift) < f.d) f.shift++;
    // round-up method: floor(2^32 (2^shift - d) / d) + 1, exact for n < 2^31
    f.mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << f.shift) - f.d)) / f.d + 1);
    return f;
}

__device__ __forceinline__ void report(uint32_t *errors, uint32_t bits) {
    if (errors) atomicOr(errors, bits);
}

inline bool cache_type(int t) { return t == OFB_TYPE_BF16 || t == OFB_TYPE_F16; }
inline bool misaligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

inline int64_t cache_page_stride(const ofb_kv_cache *c) {
    return c->page_stride ? c->page_stride : (int64_t)c->n_kv_heads * c->page_size * c->head_dim;
}
// Entries a sequence can have: the table's reach, as far as an int goes.
inline int cache_reach(const ofb_kv_cache *c) {
    const int64_t n = (int64_t)c->max_pages * c->page_size;
    return n > INT32_MAX - 64 ? INT32_MAX - 64 : (int)n;
}

// Checks the cache description; sets the error text. Reads host memory only.
inline int check_cache(const ofb_kv_cache *c, const char *who) {
    if (!c || !c->k || !c->v || !c->page_table) { set_error("%s: cache, k, v or page_table is NULL", who); return OFB_EINVAL; }
    if (!cache_type(c->type)) { set_error("%s: cache type %d is not BF16/F16", who, c->type); return OFB_EUNSUPPORTED; }
    const int d = c->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256) {
        set_error("%s: head_dim %d is not 64/96/128/192/256", who, d);
        return OFB_EUNSUPPORTED;
    }
    if (c->n_kv_heads < 1 || c->n_kv_heads > 1024 || c->page_size < 1 || c->page_size > 65536 || c->n_pages < 1 ||
        c->n_seqs < 1 || c->max_pages < 1) {
        set_error("%s: cache sizes out of range (kv heads %d, page %d, pages %d, sequences %d, pages per sequence %d)", who,
                  c->n_kv_heads, c->page_size, c->n_pages, c->n_seqs, c->max_pages);
        return OFB_EINVAL;
    }
    const int64_t dense = (int64_t)c->n_kv_heads * c->page_size * d;
    if (c->page_stride && (c->page_stride < dense || c->page_stride % 8)) {
        set_error("%s: page_stride %lld is below %lld or no multiple of 8", who, (long long)c->page_stride, (long long)dense);
        return OFB_EINVAL;
    }
    if (misaligned(c->k, 16) || misaligned(c->v, 16)) { set_error("%s: k or v is not 16-byte aligned", who); return OFB_EINVAL; }
    if (misaligned(c->weight, 4) || misaligned(c->order, 4) || misaligned(c->page_table, 4) || misaligned(c->errors, 4)) {
        set_error("%s: weight, order, page_table or errors is not 4-byte aligned", who);
        return OFB_EINVAL;
    }
    return OFB_OK;
}

inline size_t type_size(int t) { return t == OFB_TYPE_F32 ? 4 : 2; }

}  // namespace ofb
