// A caller-owned paged int8 KV cache as the row operators see it (rows into
// pages, attention over them), the element types of their inputs and outputs,
// and the checks every entry point makes.  The page layout is kv.cuh's.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv.cuh"

namespace ndl {

struct PagedCache {
    const int32_t *page_table;  // [slots][max_pages]
    uint8_t *pool;
    long long page_bytes;
    int slots, max_pages, num_pages;
    int layer, heads;  // heads: kv heads per layer
    int *status;
};

inline size_t type_bytes(int type) { return type == NDL_TYPE_F32 ? 4 : 2; }

// The cache part of an entry point's argument checks.
int check_cache(const int32_t *page_table, int slots, int max_pages, const void *pool, size_t page_bytes,
                int num_pages, int layer, int heads);
// A row-major operand [rows][heads][64] with `stride` elements between rows:
// 16-byte aligned rows that do not overlap.
int check_rows(const char *name, const void *p, int type, int heads, long long stride);
// An attention entry point's operands (attention_split.cu).
int check_attention(const void *q, long long q_stride, const void *out, long long out_stride, int type, int rows,
                    int heads, int kv_heads, float scale, int window);

#ifdef __CUDACC__
// Runs `f` with a value of the element type.
template <class F>
int with_type(int type, F &&f) {
    if (type == NDL_TYPE_F32) return f(float{});
    if (type == NDL_TYPE_F16) return f(__half{});
    return f(__nv_bfloat16{});
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (__is_same(T, __half)) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

// Page `index` of a slot, or -1 where the table has none in the pool.  The
// slot is in range; an index past the table has no page.
__device__ __forceinline__ int cache_page(const PagedCache &c, int slot, int index) {
    const int page = index < c.max_pages ? c.page_table[(size_t)slot * c.max_pages + index] : -1;
    return page >= 0 && page < c.num_pages ? page : -1;
}
__device__ __forceinline__ uint8_t *cache_record(const PagedCache &c, int page, int head) {
    return c.pool + (size_t)page * c.page_bytes + kv_block_offset(c.layer, head, c.heads);
}
#endif

}  // namespace ndl
