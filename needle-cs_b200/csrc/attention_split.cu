// Attention of single tokens over the paged int8 cache.
#include "attention_row.cuh"

namespace ndl {

struct SplitArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int32_t *row_slot, *row_len;
    int rows, heads, window;
    float scale;
    PagedCache c;
};

template <class T>
__global__ void __launch_bounds__(128) attention_split_kernel(SplitArgs a) {
    __shared__ float q[4][64];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + w;
    if (item >= (long long)a.rows * a.heads) return;
    const int row = (int)(item / a.heads), head = (int)(item % a.heads);
    const T *src = static_cast<const T *>(a.q) + (size_t)row * a.q_stride + head * 64;
    q[w][lane] = to_float(src[lane]) * a.scale;
    q[w][lane + 32] = to_float(src[lane + 32]) * a.scale;
    __syncwarp();
    const int slot = a.row_slot[row], len = a.row_len[row];
    bool ok = slot >= 0 && slot < a.c.slots && len >= 0 && len <= a.c.max_pages * 64;
    float o0, o1;
    if (ok)
        ok = attend_row(a.c, slot, head / (a.heads / a.c.heads), a.window ? max(0, len - a.window) : 0, len, q[w], o0,
                        o1, lane);
    if (!ok) {
        if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        o0 = o1 = __int_as_float(0x7fc00000);
    }
    T *dst = static_cast<T *>(a.out) + (size_t)row * a.out_stride + head * 64;
    dst[lane] = from_float<T>(o0);
    dst[lane + 32] = from_float<T>(o1);
}

int check_attention(const void *q, long long q_stride, const void *out, long long out_stride, int type, int rows,
                    int heads, int kv_heads, float scale, int window) {
    NDL_REQUIRE(type >= NDL_TYPE_F32 && type <= NDL_TYPE_BF16, "unknown element type %d", type);
    NDL_REQUIRE(heads >= 1 && heads % kv_heads == 0, "%d query heads over %d kv heads", heads, kv_heads);
    NDL_REQUIRE((long long)rows * heads <= 0x7FFFFFFFLL, "%d rows of %d heads: too many", rows, heads);
    NDL_REQUIRE(isfinite(scale) && scale > 0.0f, "scale %g is not a positive number", scale);
    NDL_REQUIRE(window >= 0, "window %d", window);
    int rc = check_rows("q", q, type, heads, q_stride);
    return rc == NDL_OK ? check_rows("out", out, type, heads, out_stride) : rc;
}

}  // namespace ndl

using namespace ndl;

extern "C" NDL_API size_t ndl_attention_split_workspace(int rows, int heads, int kv_heads, int max_pages) { return 0; }

extern "C" NDL_API int ndl_attention_split(const void *q, long long q_stride, int type, const int32_t *row_slot,
                                           const int32_t *row_len, int rows, int heads, int kv_heads, float scale,
                                           int window, const int32_t *page_table, int slots, int max_pages,
                                           const uint8_t *pool, size_t page_bytes, int num_pages, int layer, void *out,
                                           long long out_stride, void *workspace, size_t workspace_bytes, int *status,
                                           void *stream) {
    NDL_REQUIRE(rows >= 0, "bad row count %d", rows);
    int rc = check_cache(page_table, slots, max_pages, pool, page_bytes, num_pages, layer, kv_heads);
    if (rc != NDL_OK || rows == 0) return rc;
    NDL_REQUIRE(row_slot && row_len, "null pointer");
    rc = check_attention(q, q_stride, out, out_stride, type, rows, heads, kv_heads, scale, window);
    if (rc != NDL_OK) return rc;
    const size_t need = ndl_attention_split_workspace(rows, heads, kv_heads, max_pages);
    NDL_REQUIRE(aligned(workspace, 16) && (need == 0 || (workspace && workspace_bytes >= need)),
                "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    SplitArgs a{q, out, q_stride, out_stride, row_slot, row_len, rows, heads, window, scale,
                {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                 kv_heads, status}};
    return with_type(type, [&](auto t) {
        attention_split_kernel<decltype(t)>
            <<<(unsigned)(((long long)rows * heads + 3) / 4), 128, 0, (cudaStream_t)stream>>>(a);
        return check_launch("attention_split");
    });
}
