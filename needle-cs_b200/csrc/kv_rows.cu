// Rows of keys and values into and out of the paged int8 cache.
//
// Append: per (row, kv head) the quantizer the engine's own KV write applies
// (QuantizeInt8 of 64 values: scale = max|x| / 127, 1 for a zero vector,
// code = round_half_even(x * (1 / scale)) clamped), for inputs of 32 or 16
// bits; the codes and scales it stores are those ndl_quantize_rows gives for
// the same 64 values.  Gather: code * scale, the values the pages stand for.
//
// Both are bound by memory, and by how the pages scatter a row: its 64 value
// bytes lie 64 bytes apart, its keys in 16 words.  So rows of a block that
// follow one another inside a 16-position chunk of a page (a run) go to one
// warp a head: a lane holds 32 dims of one position; keys change hands between
// positions 8 apart and move as 16-byte chunks, values turn around in shared
// memory (4x4 bytes by permutes) and move 4 positions of a dim at a time.
// Other rows, as a decode step has them, go 16 to a warp, each by its words
// and bytes.
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

struct KvRowsArgs {
    const void *k, *v;
    void *k_out, *v_out;
    long long k_stride, v_stride;
    const int32_t *row_slot, *row_pos;
    int rows, block_rows;
    PagedCache c;
};

constexpr int kRowWarps = 2, kRowThreads = 32 * kRowWarps;
constexpr int kBlockRows = 32;           // rows of a block, at most: a warp looks them over
constexpr int kChunk = 16;               // positions of a chunk: 16 bytes of a value dim
constexpr int kShortRun = 3;             // rows from which a run is worth a warp
constexpr int kTurnRow = kHeadDim + 4;   // a position's codes in shared memory: 17 words, so positions on different banks

struct KvRowsSmem {
    __align__(16) uint8_t turn[kRowWarps][kChunk * kTurnRow];
    uint8_t *rec[kBlockRows];  // the row's record of head 0, null for a padding or bad row
    int place[kBlockRows];     // its position in the page
    int bad[kBlockRows];
    int runs[kBlockRows], singles[kBlockRows];  // runs: first row | length << 8
    int run_count, single_count;
};

// The block's rows: where they go, its runs and its single rows.
__device__ __forceinline__ void kv_rows_block(const KvRowsArgs &a, KvRowsSmem &s, int first) {
    if (threadIdx.x < 32) {
        const int n = min(a.block_rows, a.rows - first), i = threadIdx.x;
        uint8_t *rec = nullptr;
        int place = 0, bad = 0;
        if (i < n) {
            const int pos = a.row_pos[first + i], slot = a.row_slot[first + i];
            if (pos >= 0) {
                const int page = slot >= 0 && slot < a.c.slots ? cache_page(a.c, slot, pos / kPagePositions) : -1;
                bad = page < 0;
                place = pos % kPagePositions;
                if (!bad) rec = cache_record(a.c, page, 0);
                else if (a.c.status) atomicOr(a.c.status, kStatusBadPage);
            }
            s.rec[i] = rec, s.place[i] = place, s.bad[i] = bad;
        }
        const unsigned long long before = __shfl_up_sync(0xffffffffu, (unsigned long long)rec, 1);
        const int before_place = __shfl_up_sync(0xffffffffu, place, 1);
        const bool starts = i < n && !(i > 0 && rec && (unsigned long long)rec == before && place == before_place + 1 &&
                                       (place & (kChunk - 1)) != 0);
        const unsigned mask = __ballot_sync(0xffffffffu, starts);
        const unsigned upto = mask & (0xFFFFFFFFu >> (31 - i)), behind = i < 31 ? mask >> (i + 1) : 0;
        const int start = 31 - __clz((int)upto), end = behind ? i + __ffs((int)behind) : n;
        const bool in_run = i < n && rec && end - start >= kShortRun;
        const unsigned runs = __ballot_sync(0xffffffffu, starts && in_run);
        const unsigned singles = __ballot_sync(0xffffffffu, i < n && !in_run);
        const unsigned below = (1u << i) - 1;
        if (starts && in_run) s.runs[__popc(runs & below)] = i | (end - start) << 8;
        if (i < n && !in_run) s.singles[__popc(singles & below)] = i;
        if (i == 0) s.run_count = __popc(runs), s.single_count = __popc(singles);
    }
    __syncthreads();
}

// 4x4 bytes turned around: word j of the result holds byte j of each word.
__device__ __forceinline__ void turn4(uint32_t (&w)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
    w[0] = __byte_perm(a, b, 0x5410), w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(c, d, 0x5410), w[3] = __byte_perm(c, d, 0x7632);
}

// Lane (position r = lane & 15 of the chunk, half = lane >> 4): dims 32 half .. + 31, word c of them at w[c].  In the
// pages, chunk (row & 7, column t) of a 32-dim step holds words (r, t), (r + 8, t), (r, t + 4), (r + 8, t + 4); the lane
// of r < 8 moves columns 0 and 1 of both positions, that of r + 8 columns 2 and 3.
__device__ __forceinline__ void swap_columns(uint32_t (&w)[8], bool upper) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int give_low = (i >> 1) * 4 + (i & 1), give_high = give_low + 2;  // words of columns 0, 1 / 2, 3
        const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[give_low] : w[give_high], 8);
        if (upper) w[give_low] = got;
        else w[give_high] = got;
    }
}

template <class T>
__device__ __forceinline__ void load32(const T *p, float (&x)[32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(p + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + i);
            const T *h = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int j = 0; j < 8; j++) x[i + j] = to_float(h[j]);
        }
    }
}
template <class T>
__device__ __forceinline__ void store32(T *p, const float (&x)[32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            alignas(16) T h[8];
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = from_float<T>(x[i + j]);
            *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(h);
        }
    }
}

// The codes of a lane's 32 dims and its position's scale (the partner holds the other 32).  Adding 1.5 * 2^23 rounds to
// an integer, ties to even, and leaves it in the low byte; a NaN becomes -128 as the quantizer's clamp makes it.
__device__ __forceinline__ float quantize32(const float (&x)[32], uint32_t (&w)[8]) {
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; i++) peak = fmaxf(peak, fabsf(x[i]));
    peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 16));
    const float scale = peak > 0.0f ? __fdiv_rn(peak, 127.0f) : 1.0f;
    const float inverse = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int c = 0; c < 8; c++) {
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            b[j] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x[4 * c + j], inverse), -128.0f), 127.0f), 12582912.0f));
        w[c] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    return scale;
}

// A warp's share of a block: run i of the block, then 16 single rows a task.
struct KvTask {
    int row;              // this lane's row of the block
    bool mine;            // it has one
    uint8_t *rec;         // its record (null: padding or bad)
    int place;            // its position in the page
    bool run;             // the warp's rows are a run,
    int from, to, chunk;  // positions from .. to - 1 of a 16-position chunk
};
__device__ __forceinline__ KvTask kv_task(const KvRowsSmem &s, int i, int head, int r) {
    KvTask t;
    t.run = i < s.run_count;
    if (t.run) {
        const int row0 = s.runs[i] & 0xFF, n = s.runs[i] >> 8, place = s.place[row0];
        t.from = place & (kChunk - 1), t.to = t.from + n, t.chunk = place >> 4;
        t.mine = r >= t.from && r < t.to;
        t.row = row0 + (t.mine ? r - t.from : 0);
        t.rec = s.rec[row0] + (size_t)head * kKvBlockBytes;
        t.place = t.chunk * kChunk + r;
    } else {
        const int j = (i - s.run_count) * kChunk + r;
        t.mine = j < s.single_count;
        t.row = s.singles[t.mine ? j : 0];
        t.rec = s.rec[t.row];
        if (t.rec) t.rec += (size_t)head * kKvBlockBytes;
        t.place = s.place[t.row];
        t.from = t.to = t.chunk = 0;
    }
    return t;
}
__device__ __forceinline__ int kv_tasks(const KvRowsSmem &s) {
    return s.run_count + (s.single_count + kChunk - 1) / kChunk;
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 12) kv_append_kernel(KvRowsArgs a) {
    __shared__ KvRowsSmem s;
    const int first = blockIdx.x * a.block_rows, head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
    kv_rows_block(a, s, first);
    const int tasks = kv_tasks(s);
    for (int i = warp; i < tasks; i += kRowWarps) {
        const KvTask t = kv_task(s, i, head, r);
        const size_t at = first + t.row;
        float x[32];
        uint32_t w[8];
        load32(static_cast<const T *>(a.k) + at * a.k_stride + head * kHeadDim + 32 * half, x);
        const float ks = quantize32(x, w);
        load32(static_cast<const T *>(a.v) + at * a.v_stride + head * kHeadDim + 32 * half, x);
        const bool writes = t.mine && t.rec;
        if (writes && half == 0) reinterpret_cast<float *>(t.rec + kKScaleOffset)[k_scale_index(t.place)] = ks;
        if (t.run) {
            const bool partner = (r ^ 8) >= t.from && (r ^ 8) < t.to;
            swap_columns(w, r >= 8);
            // words (position, column) and (position + 8, column) of columns t0 and t0 + 1
            const int t0 = r >= 8 ? 2 : 0;
            const bool low = r >= 8 ? partner : t.mine, high = r >= 8 ? t.mine : partner;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t *dst = reinterpret_cast<uint32_t *>(t.rec + t.chunk * 1024 + half * 512 + ((r & 7) * 4 + t0 + j) * 16);
                // own words of the column, and the partner's in the place of those given away
                const uint32_t o0 = r >= 8 ? w[2 + j] : w[j], o1 = r >= 8 ? w[6 + j] : w[4 + j];
                const uint32_t p0 = r >= 8 ? w[j] : w[2 + j], p1 = r >= 8 ? w[4 + j] : w[6 + j];
                const uint32_t a0 = r >= 8 ? p0 : o0, a1 = r >= 8 ? p1 : o1, b0 = r >= 8 ? o0 : p0, b1 = r >= 8 ? o1 : p1;
                if (low && high) {
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(a0, b0, a1, b1);
                } else {
                    if (low) dst[0] = a0, dst[2] = a1;
                    if (high) dst[1] = b0, dst[3] = b1;
                }
            }
        } else if (writes) {
#pragma unroll
            for (int c = 0; c < 8; c++) *reinterpret_cast<uint32_t *>(t.rec + k_byte(t.place, 32 * half + 4 * c)) = w[c];
        }
        const float vs = quantize32(x, w);
        if (writes && half == 0) reinterpret_cast<float *>(t.rec + kVScaleOffset)[v_scale_index(t.place)] = vs;
        if (t.run) {
            uint32_t *turn = reinterpret_cast<uint32_t *>(s.turn[warp]);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; c++) turn[r * (kTurnRow / 4) + half * 8 + c] = w[c];
            __syncwarp();
            // lane -> positions 4 q .. of dims 4 c ..
            const int q = lane & 3;
            if (4 * q + 4 > t.from && 4 * q < t.to) {
                const bool all = 4 * q >= t.from && 4 * q + 4 <= t.to;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int c = (lane >> 2) + 8 * h;
                    uint32_t b[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) b[j] = turn[(4 * q + j) * (kTurnRow / 4) + c];
                    turn4(b);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint8_t *dst = t.rec + v_byte(t.chunk * kChunk + 4 * q, 4 * c + j);
                        if (all) *reinterpret_cast<uint32_t *>(dst) = b[j];
                        else
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (4 * q + e >= t.from && 4 * q + e < t.to) dst[e] = (uint8_t)(b[j] >> (8 * e));
                    }
                }
            }
        } else if (writes) {
#pragma unroll
            for (int j = 0; j < 32; j++) t.rec[v_byte(t.place, 32 * half + j)] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, 12) kv_gather_kernel(KvRowsArgs a) {
    __shared__ KvRowsSmem s;
    const int first = blockIdx.x * a.block_rows, head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane & 15, half = lane >> 4;
    kv_rows_block(a, s, first);
    const int tasks = kv_tasks(s);
    for (int i = warp; i < tasks; i += kRowWarps) {
        const KvTask t = kv_task(s, i, head, r);
        const size_t at = first + t.row;
        T *k = static_cast<T *>(a.k_out) + at * a.k_stride + head * kHeadDim + 32 * half;
        T *v = static_cast<T *>(a.v_out) + at * a.v_stride + head * kHeadDim + 32 * half;
        uint32_t kw[8] = {}, vw[8] = {};
        float ks = 0.0f, vs = 0.0f;
        if (t.rec) {
            ks = __ldg(reinterpret_cast<const float *>(t.rec + kKScaleOffset) + k_scale_index(t.place));
            vs = __ldg(reinterpret_cast<const float *>(t.rec + kVScaleOffset) + v_scale_index(t.place));
        } else if (s.bad[t.row]) {  // NaN; a padding row gives zeros
            ks = vs = __int_as_float(0x7fc00000);
        }
        if (t.run) {
            const int t0 = r >= 8 ? 2 : 0;
            uint4 dim[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint4 c =
                    __ldg(reinterpret_cast<const uint4 *>(t.rec + t.chunk * 1024 + half * 512 + ((r & 7) * 4 + t0 + j) * 16));
                dim[j] = __ldg(reinterpret_cast<const uint4 *>(t.rec + v_byte(t.chunk * kChunk, lane + 32 * j)));
                // own words of columns t0 + j in their place, the partner's in the place of what it will give
                const uint32_t o0 = r >= 8 ? c.y : c.x, o1 = r >= 8 ? c.w : c.z, p0 = r >= 8 ? c.x : c.y, p1 = r >= 8 ? c.z : c.w;
                kw[j] = r >= 8 ? p0 : o0, kw[4 + j] = r >= 8 ? p1 : o1;
                kw[2 + j] = r >= 8 ? o0 : p0, kw[6 + j] = r >= 8 ? o1 : p1;
            }
            swap_columns(kw, r >= 8);
            // values: dims as rows of 16 bytes, turned around to positions as rows
            uint32_t *turn = reinterpret_cast<uint32_t *>(s.turn[warp]);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 2; j++) *reinterpret_cast<uint4 *>(turn + (lane + 32 * j) * 4) = dim[j];
            __syncwarp();
            const int q = lane & 3;
            uint32_t b[2][4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int j = 0; j < 4; j++) b[h][j] = turn[(4 * ((lane >> 2) + 8 * h) + j) * 4 + q];
                turn4(b[h]);
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < 4; j++) turn[(4 * q + j) * (kTurnRow / 4) + (lane >> 2) + 8 * h] = b[h][j];
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 8; c++) vw[c] = turn[r * (kTurnRow / 4) + half * 8 + c];
        } else if (t.rec) {
#pragma unroll
            for (int c = 0; c < 8; c++)
                kw[c] = __ldg(reinterpret_cast<const uint32_t *>(t.rec + k_byte(t.place, 32 * half + 4 * c)));
#pragma unroll
            for (int j = 0; j < 32; j++) vw[j >> 2] |= (uint32_t)__ldg(t.rec + v_byte(t.place, 32 * half + j)) << (8 * (j & 3));
        }
        if (!t.mine) continue;
        float x[32];
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = __fmul_rn((float)(int8_t)(uint8_t)(kw[j >> 2] >> (8 * (j & 3))), ks);
        store32(k, x);
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = __fmul_rn((float)(int8_t)(uint8_t)(vw[j >> 2] >> (8 * (j & 3))), vs);
        store32(v, x);
    }
}

// Rows a block, whose CTAs (one a head) are small because single rows cost an SM's load/store unit a clock a byte of
// values: 32 where that leaves every SM two blocks, else 16, a warp's share of single rows.
static int block_rows(int rows, int heads) {
    return (long long)((rows + kBlockRows - 1) / kBlockRows) * heads >= 2 * 148 ? kBlockRows : kChunk;
}

static int check_kv_rows(int type, int rows, int heads, const void *k, long long k_stride, const void *v,
                         long long v_stride, const int32_t *row_slot, const int32_t *row_pos) {
    NDL_REQUIRE(type >= NDL_TYPE_F32 && type <= NDL_TYPE_BF16, "unknown element type %d", type);
    NDL_REQUIRE(row_slot && row_pos, "null pointer");
    int rc = check_rows("k", k, type, heads, k_stride);
    if (rc == NDL_OK) rc = check_rows("v", v, type, heads, v_stride);
    if (rc != NDL_OK) return rc;
    NDL_REQUIRE((long long)rows * heads <= 0x7FFFFFFFLL && heads <= 65535, "%d rows of %d heads: too many", rows, heads);
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
    KvRowsArgs a{k, v, nullptr, nullptr, k_stride, v_stride, row_slot, row_pos, rows, block_rows(rows, kv_heads),
                 {page_table, pool, (long long)page_bytes, slots, max_pages, num_pages, layer, kv_heads, status}};
    const dim3 grid((rows + a.block_rows - 1) / a.block_rows, kv_heads);
    return with_type(type, [&](auto t) {
        kv_append_kernel<decltype(t)><<<grid, kRowThreads, 0, (cudaStream_t)stream>>>(a);
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
    KvRowsArgs a{nullptr, nullptr, k, v, k_stride, v_stride, row_slot, row_pos, rows, block_rows(rows, kv_heads),
                 {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                  kv_heads, status}};
    const dim3 grid((rows + a.block_rows - 1) / a.block_rows, kv_heads);
    return with_type(type, [&](auto t) {
        kv_gather_kernel<decltype(t)><<<grid, kRowThreads, 0, (cudaStream_t)stream>>>(a);
        return check_launch("kv_gather");
    });
}
