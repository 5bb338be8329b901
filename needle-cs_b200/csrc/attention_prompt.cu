// Attention of whole prompts over the paged int8 cache.
#include "attention_row.cuh"

namespace ndl {

struct PromptArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int32_t *seq_rows, *seq_slot, *seq_pos;
    int rows, sequences, heads, window;
    float scale;
    PagedCache c;
};

template <class T>
__global__ void __launch_bounds__(128) attention_prompt_kernel(PromptArgs a) {
    __shared__ float q[4][64];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + w;
    if (item >= (long long)a.rows * a.heads) return;
    const int row = (int)(item / a.heads), head = (int)(item % a.heads);
    int seq = -1;
    for (int s = 0; s < a.sequences; s++) {
        const int b = a.seq_rows[s], e = a.seq_rows[s + 1];
        if (b < 0 || e < b || e > a.rows) {
            if (item == 0 && lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        } else if (b <= row && row < e) {
            seq = s;
        }
    }
    if (seq < 0) return;  // in no sequence
    const T *src = static_cast<const T *>(a.q) + (size_t)row * a.q_stride + head * 64;
    q[w][lane] = to_float(src[lane]) * a.scale;
    q[w][lane + 32] = to_float(src[lane + 32]) * a.scale;
    __syncwarp();
    const int slot = a.seq_slot[seq], start = a.seq_pos[seq], n = a.seq_rows[seq + 1] - a.seq_rows[seq];
    bool ok = slot >= 0 && slot < a.c.slots && start >= 0 && (long long)start + n <= (long long)a.c.max_pages * 64;
    float o0, o1;
    if (ok) {
        const int len = start + row - a.seq_rows[seq] + 1;
        ok = attend_row(a.c, slot, head / (a.heads / a.c.heads), a.window ? max(0, len - a.window) : 0, len, q[w], o0,
                        o1, lane);
    }
    if (!ok) {
        if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        o0 = o1 = __int_as_float(0x7fc00000);
    }
    T *dst = static_cast<T *>(a.out) + (size_t)row * a.out_stride + head * 64;
    dst[lane] = from_float<T>(o0);
    dst[lane + 32] = from_float<T>(o1);
}

}  // namespace ndl

using namespace ndl;

extern "C" NDL_API int ndl_attention_prompt(const void *q, long long q_stride, int type, const int32_t *seq_rows,
                                            const int32_t *seq_slot, const int32_t *seq_pos, int sequences, int rows,
                                            int heads, int kv_heads, float scale, int window,
                                            const int32_t *page_table, int slots, int max_pages, const uint8_t *pool,
                                            size_t page_bytes, int num_pages, int layer, void *out,
                                            long long out_stride, int *status, void *stream) {
    NDL_REQUIRE(rows >= 0 && sequences >= 0, "bad row count %d or sequence count %d", rows, sequences);
    int rc = check_cache(page_table, slots, max_pages, pool, page_bytes, num_pages, layer, kv_heads);
    if (rc != NDL_OK || rows == 0 || sequences == 0) return rc;
    NDL_REQUIRE(seq_rows && seq_slot && seq_pos, "null pointer");
    rc = check_attention(q, q_stride, out, out_stride, type, rows, heads, kv_heads, scale, window);
    if (rc != NDL_OK) return rc;
    PromptArgs a{q, out, q_stride, out_stride, seq_rows, seq_slot, seq_pos, rows, sequences, heads, window, scale,
                 {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                  kv_heads, status}};
    return with_type(type, [&](auto t) {
        attention_prompt_kernel<decltype(t)>
            <<<(unsigned)(((long long)rows * heads + 3) / 4), 128, 0, (cudaStream_t)stream>>>(a);
        return check_launch("attention_prompt");
    });
}
