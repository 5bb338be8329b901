// Rows of keys and values into and out of the paged int8 cache.
//
// Append: per (row, kv head) the quantizer the engine's own KV write applies
// (QuantizeInt8 of 64 values: scale = max|x| / 127, 1 for a zero vector,
// code = round_half_even(x * (1 / scale)) clamped), for inputs of 32 or 16
// bits; the codes and scales it stores are those ndl_quantize_rows gives for
// the same 64 values.  Gather: code * scale, the values the pages stand for.
#include "paged.cuh"

namespace ndl {

int check_cache(const int32_t *page_table, int slots, int max_pages, const void *pool, size_t page_bytes,
                int num_pages, int layer, int heads) {
    NDL_REQUIRE(heads >= 1 && slots >= 1 && max_pages >= 1 && num_pages >= 1 && layer >= 0, "bad cache geometry");
    NDL_REQUIRE(page_table && pool, "null pointer");
    NDL_REQUIRE((long long)max_pages * kPagePositions <= 0x7FFFFFFF, "%d pages a slot: more positions than an int",
                max_pages);
    NDL_REQUIRE(page_bytes % 16 == 0 && page_bytes >= kv_block_offset(layer, heads - 1, heads) + kKvBlockBytes,
                "page_bytes %zu cannot hold layer %d of %d heads", page_bytes, layer, heads);
    NDL_REQUIRE(aligned(pool, 16) && aligned(page_table, 4), "misaligned pointer");
    return NDL_OK;
}

int check_rows(const char *name, const void *p, int type, int heads, long long stride) {
    NDL_REQUIRE(p, "%s: null pointer", name);
    const long long width = (long long)heads * kHeadDim, per16 = 16 / (long long)type_bytes(type);
    NDL_REQUIRE(stride >= width && stride % per16 == 0, "%s: row stride %lld (at least %lld, a multiple of %lld)", name,
                stride, width, per16);
    NDL_REQUIRE(aligned(p, 16), "%s: misaligned pointer", name);
    return NDL_OK;
}

__device__ __forceinline__ float row_warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ uint8_t row_code(float x, float inverse) {
    const float r = rintf(__fmul_rn(x, inverse));
    return (uint8_t)(int8_t)(int)fminf(fmaxf(r, -128.0f), 127.0f);
}

struct KvRowsArgs {
    const void *k, *v;
    void *k_out, *v_out;
    long long k_stride, v_stride;
    const int32_t *row_slot, *row_pos;
    int rows;
    PagedCache c;
};

// Record of a row's position in head `head`, null for a padding row or a bad
// one (which sets the status).
__device__ __forceinline__ uint8_t *kv_row_record(const KvRowsArgs &a, int row, int head, int lane, int &place,
                                                  bool &padding) {
    const int pos = a.row_pos[row], slot = a.row_slot[row];
    padding = pos < 0;
    if (padding) return nullptr;
    const int page = slot >= 0 && slot < a.c.slots ? cache_page(a.c, slot, pos / kPagePositions) : -1;
    if (page < 0) {
        if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        return nullptr;
    }
    place = pos % kPagePositions;
    return cache_record(a.c, page, head);
}

template <class T>
__global__ void __launch_bounds__(256) kv_append_kernel(KvRowsArgs a) {
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (warp >= (long long)a.rows * a.c.heads) return;
    const int row = (int)(warp / a.c.heads), head = (int)(warp % a.c.heads);
    int place = 0;
    bool padding;
    uint8_t *rec = kv_row_record(a, row, head, lane, place, padding);
    if (!rec) return;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        const T *src = static_cast<const T *>(which ? a.v : a.k) + (size_t)row * (which ? a.v_stride : a.k_stride) +
                       head * kHeadDim;
        const float lo = to_float(src[lane]), hi = to_float(src[lane + 32]);
        const float peak = row_warp_max(fmaxf(fabsf(lo), fabsf(hi)));
        const float scale = peak > 0.0f ? __fdiv_rn(peak, 127.0f) : 1.0f;
        const float inverse = __fdiv_rn(1.0f, scale);
        rec[which ? v_byte(place, lane) : k_byte(place, lane)] = row_code(lo, inverse);
        rec[which ? v_byte(place, lane + 32) : k_byte(place, lane + 32)] = row_code(hi, inverse);
        if (lane == 0) {
            if (which) reinterpret_cast<float *>(rec + kVScaleOffset)[v_scale_index(place)] = scale;
            else reinterpret_cast<float *>(rec + kKScaleOffset)[k_scale_index(place)] = scale;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(256) kv_gather_kernel(KvRowsArgs a) {
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (warp >= (long long)a.rows * a.c.heads) return;
    const int row = (int)(warp / a.c.heads), head = (int)(warp % a.c.heads);
    int place = 0;
    bool padding;
    const uint8_t *rec = kv_row_record(a, row, head, lane, place, padding);
#pragma unroll
    for (int which = 0; which < 2; which++) {
        T *dst = static_cast<T *>(which ? a.v_out : a.k_out) + (size_t)row * (which ? a.v_stride : a.k_stride) +
                 head * kHeadDim;
        float lo = 0.0f, hi = 0.0f;
        if (rec) {
            const float scale = which ? reinterpret_cast<const float *>(rec + kVScaleOffset)[v_scale_index(place)]
                                      : reinterpret_cast<const float *>(rec + kKScaleOffset)[k_scale_index(place)];
            lo = (float)(int8_t)rec[which ? v_byte(place, lane) : k_byte(place, lane)] * scale;
            hi = (float)(int8_t)rec[which ? v_byte(place, lane + 32) : k_byte(place, lane + 32)] * scale;
        } else if (!padding) {
            lo = hi = __int_as_float(0x7fc00000);
        }
        dst[lane] = from_float<T>(lo);
        dst[lane + 32] = from_float<T>(hi);
    }
}

static int check_kv_rows(int type, int rows, int heads, const void *k, long long k_stride, const void *v,
                         long long v_stride, const int32_t *row_slot, const int32_t *row_pos) {
    NDL_REQUIRE(type >= NDL_TYPE_F32 && type <= NDL_TYPE_BF16, "unknown element type %d", type);
    NDL_REQUIRE(row_slot && row_pos, "null pointer");
    int rc = check_rows("k", k, type, heads, k_stride);
    if (rc == NDL_OK) rc = check_rows("v", v, type, heads, v_stride);
    if (rc != NDL_OK) return rc;
    NDL_REQUIRE((long long)rows * heads <= 0x7FFFFFFFLL, "%d rows of %d heads: too many", rows, heads);
    return NDL_OK;
}

}  // namespace ndl

using namespace ndl;

extern "C" NDL_API int ndl_kv_append(const void *k, long long k_stride, const void *v, long long v_stride, int type,
                                     const int32_t *row_slot, const int32_t *row_pos, int rows, int kv_heads,
                                     const int32_t *page_table, int slots, int max_pages, uint8_t *pool,
                                     size_t page_bytes, int num_pages, int layer, int *status, void *stream) {
    NDL_REQUIRE(rows >= 0, "bad row count %d", rows);
    int rc = check_cache(page_table, slots, max_pages, pool, page_bytes, num_pages, layer, kv_heads);
    if (rc != NDL_OK || rows == 0) return rc;
    rc = check_kv_rows(type, rows, kv_heads, k, k_stride, v, v_stride, row_slot, row_pos);
    if (rc != NDL_OK) return rc;
    KvRowsArgs a{k, v, nullptr, nullptr, k_stride, v_stride, row_slot, row_pos, rows,
                 {page_table, pool, (long long)page_bytes, slots, max_pages, num_pages, layer, kv_heads, status}};
    const unsigned blocks = (unsigned)(((long long)rows * kv_heads + 7) / 8);
    return with_type(type, [&](auto t) {
        kv_append_kernel<decltype(t)><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
        return check_launch("kv_append");
    });
}

extern "C" NDL_API int ndl_kv_gather(const int32_t *row_slot, const int32_t *row_pos, int rows, int kv_heads,
                                     const int32_t *page_table, int slots, int max_pages, const uint8_t *pool,
                                     size_t page_bytes, int num_pages, int layer, void *k, long long k_stride,
                                     void *v, long long v_stride, int type, int *status, void *stream) {
    NDL_REQUIRE(rows >= 0, "bad row count %d", rows);
    int rc = check_cache(page_table, slots, max_pages, pool, page_bytes, num_pages, layer, kv_heads);
    if (rc != NDL_OK || rows == 0) return rc;
    rc = check_kv_rows(type, rows, kv_heads, k, k_stride, v, v_stride, row_slot, row_pos);
    if (rc != NDL_OK) return rc;
    KvRowsArgs a{nullptr, nullptr, k, v, k_stride, v_stride, row_slot, row_pos, rows,
                 {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                  kv_heads, status}};
    const unsigned blocks = (unsigned)(((long long)rows * kv_heads + 7) / 8);
    return with_type(type, [&](auto t) {
        kv_gather_kernel<decltype(t)><<<blocks, 256, 0, (cudaStream_t)stream>>>(a);
        return check_launch("kv_gather");
    });
}
