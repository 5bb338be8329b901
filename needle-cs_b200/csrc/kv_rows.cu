// Rows of keys and values into and out of the paged int8 cache.
//
// Append: per (row, kv head) the quantizer the engine's own KV write applies
// (QuantizeInt8 of 64 values: scale = max|x| / 127, 1 for a zero vector,
// code = round_half_even(x * (1 / scale)) clamped), for inputs of 32 or 16
// bits; the codes and scales it stores are those ndl_quantize_rows gives for
// the same 64 values.  Gather: code * scale, the values the pages stand for.
//
// Both are bound by memory, and by how the pages scatter a row: its 64 value
// bytes lie 64 bytes apart, its keys in 16 words.  So a warp takes up to 16
// rows of a head, eight lanes a row where rows are read or written (four rows
// an access), and turns their codes around in shared memory.  Rows that follow
// one another inside a 16-position chunk of a page (a run) then move their keys
// as 16-byte chunks and their values 4 positions of a dim at a time (4x4 bytes
// by permutes); others, as a decode step has them, go by words and bytes.
// 16384 rows of 8 heads, bf16, all but 1243 in runs: 53 us written and read back
// (floor 16; 109 when every row went by words and bytes).  A CTA waits for its
// rows' places, then for the rows; the single rows' value bytes take a sector
// each, read and written whole (40 MB, some 9 us at the end).  64 rows, fp32: 8
// us each way, a launch and three dependent trips to memory.
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
// CTAs an SM: waits for memory fill a CTA's time, so as many as registers allow, short of spills (16384 rows of runs, bf16,
// with 10, 12, 14 and 16: append 22.3, 21.5, 20.8 and 20.9 us, gather 16.2, 16.3, 15.0 and 14.8).
template <class T>
constexpr int kAppendCtas = sizeof(T) == 4 ? 10 : 12;
template <class T>
constexpr int kGatherCtas = sizeof(T) == 4 ? 10 : 16;
constexpr int kBlockRows = 32;           // rows of a block, at most
constexpr int kChunk = 16;               // positions of a chunk: 16 bytes of a value dim
constexpr int kSeenRows = kBlockRows + kChunk;  // and of the runs that start in it: a run is the block's it starts in
constexpr int kShortRun = 3;             // rows from which a run is worth a warp
constexpr int kTurnRow = kHeadDim + 4;   // a position's codes in shared memory: 17 words, so positions on different banks

struct KvRowsSmem {
    __align__(16) uint8_t turn[kRowWarps][kChunk * kTurnRow];
    uint8_t *rec[kSeenRows];  // the row's record of head 0, null for a padding or bad row
    int place[kSeenRows];     // its position in the page
    int bad[kSeenRows];
    int runs[kBlockRows], singles[kSeenRows];  // runs: first row | length << 8
    int run_count, single_count;
};

// The block's rows: where they go, its runs and its single rows.
__device__ __forceinline__ void kv_rows_block(const KvRowsArgs &a, KvRowsSmem &s, int first) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const int own = min(a.block_rows, a.rows - first), n = min(own + kChunk, a.rows - first);
        uint8_t *rec[2] = {nullptr, nullptr};
        int place[2] = {0, 0};
        uint64_t starts = 0;
        // the row before the block and, behind, the rows its last run may reach
        const auto look = [&](int i, uint8_t *&rec, int &place, bool keep) {
            const int pos = a.row_pos[first + i], slot = a.row_slot[first + i];
            int bad = 0;
            if (pos >= 0) {
                const int page = slot >= 0 && slot < a.c.slots ? cache_page(a.c, slot, pos / kPagePositions) : -1;
                bad = page < 0;
                place = pos % kPagePositions;
                if (!bad) rec = cache_record(a.c, page, 0);
                else if (keep && i < own && a.c.status) atomicOr(a.c.status, kStatusBadPage);
            }
            if (keep) s.rec[i] = rec, s.place[i] = place, s.bad[i] = bad;
        };
        uint8_t *before = nullptr;
        int before_place = 0;
        if (lane == 0 && first > 0) look(-1, before, before_place, false);
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (lane + 32 * h < n) look(lane + 32 * h, rec[h], place[h], true);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = lane + 32 * h;
            unsigned long long up = __shfl_up_sync(0xffffffffu, (unsigned long long)rec[h], 1);
            int up_place = __shfl_up_sync(0xffffffffu, place[h], 1);
            if (lane == 0) up = (unsigned long long)before, up_place = before_place;
            before = (uint8_t *)__shfl_sync(0xffffffffu, (unsigned long long)rec[h], 31);
            before_place = __shfl_sync(0xffffffffu, place[h], 31);
            const bool start = i < n && !(rec[h] && (unsigned long long)rec[h] == up && place[h] == up_place + 1 &&
                                          (place[h] & (kChunk - 1)) != 0);
            starts |= (uint64_t)__ballot_sync(0xffffffffu, start) << (32 * h);
        }
        const uint64_t owned = own >= 64 ? ~0ull : (1ull << own) - 1;  // rows of the block itself
        uint64_t runs = 0, singles = 0;
        int length[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = lane + 32 * h;
            const uint64_t upto = starts & owned & (~0ull >> (63 - i)), behind = i < 63 ? starts >> (i + 1) : 0;
            const int start = 63 - __clzll((long long)upto);  // -1: the run of an earlier block
            const int end = behind ? i + __ffsll((long long)behind) : n;
            // behind the block only rows of a run that starts in it
            const bool ours = i < n && start >= 0 && (i < own || !(starts >> own & (~0ull >> (63 - i + own))));
            length[h] = end - i;
            const bool in_run = ours && rec[h] && end - start >= kShortRun;
            runs |= (uint64_t)__ballot_sync(0xffffffffu, in_run && start == i) << (32 * h);
            singles |= (uint64_t)__ballot_sync(0xffffffffu, ours && !in_run) << (32 * h);
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = lane + 32 * h;
            const uint64_t below = (1ull << i) - 1;
            if (runs >> i & 1) s.runs[__popcll(runs & below)] = i | length[h] << 8;
            if (singles >> i & 1) s.singles[__popcll(singles & below)] = i;
        }
        if (lane == 0) s.run_count = __popcll(runs), s.single_count = __popcll(singles);
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

// Eight lanes a row: lane -> dims 8 (lane & 7) .. of row 4 j + (lane >> 3).
template <class T>
struct Eight {
    uint4 raw[sizeof(T) == 4 ? 2 : 1];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); i++) raw[i] = *(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ float get(int i) const { return to_float(reinterpret_cast<const T *>(raw)[i]); }
    __device__ __forceinline__ void set(int i, float x) { reinterpret_cast<T *>(raw)[i] = from_float<T>(x); }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); i++) *(reinterpret_cast<uint4 *>(p) + i) = raw[i];
    }
};

// Scales and inverses of four rows, of which the lane holds eight dims each.  The two quotients of a row are one lane's.
template <class T>
__device__ __forceinline__ void row_scales(const Eight<T> (&x)[4], int lane, float (&scale)[4], float (&inverse)[4]) {
    float peak[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        peak[j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) peak[j] = fmaxf(peak[j], fabsf(x[j].get(i)));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) peak[j] = fmaxf(peak[j], __shfl_xor_sync(0xffffffffu, peak[j], o));
    }
    const float p01 = lane & 1 ? peak[1] : peak[0], p23 = lane & 1 ? peak[3] : peak[2], mine = lane & 2 ? p23 : p01;
    const float s = mine > 0.0f ? __fdiv_rn(mine, 127.0f) : 1.0f;
    const float v = __fdiv_rn(1.0f, s);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        scale[j] = __shfl_sync(0xffffffffu, s, (lane & 24) | j);
        inverse[j] = __shfl_sync(0xffffffffu, v, (lane & 24) | j);
    }
}
// Eight codes.  Adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low byte; a NaN becomes -128
// as the quantizer's clamp makes it.
template <class T>
__device__ __forceinline__ uint2 quantize8(const Eight<T> &x, float inverse) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        b[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(x.get(i), inverse), -128.0f), 127.0f), 12582912.0f));
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}
// Eight codes times a scale (the code by the low mantissa byte of 2^23, less 2^23 + 128).
template <class T>
__device__ __forceinline__ void scale8(uint2 w, float scale, Eight<T> &x) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t u = (i < 4 ? w.x : w.y) ^ 0x80808080u;
        x.set(i, __fmul_rn(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + (i & 3))) - 8388736.0f, scale));
    }
}

// A warp's share of a block: run i of the block, then 16 single rows a task.  Its 16 places: the positions of the run's
// chunk, or one a single row.
struct KvTask {
    bool run;
    int from, to;  // places that have a row
    int row0;      // run: row of place `from`; else number of the first single row
    uint8_t *rec;  // run: its record
    int chunk;     // run: its chunk of the page
};
__device__ __forceinline__ int kv_tasks(const KvRowsSmem &s) {
    return s.run_count + (s.single_count + kChunk - 1) / kChunk;
}
__device__ __forceinline__ KvTask kv_task(const KvRowsSmem &s, int i, int head) {
    KvTask t;
    t.run = i < s.run_count;
    if (t.run) {
        t.row0 = s.runs[i] & 0xFF;
        const int place = s.place[t.row0];
        t.from = place & (kChunk - 1), t.to = t.from + (s.runs[i] >> 8), t.chunk = place >> 4;
        t.rec = s.rec[t.row0] + (size_t)head * kKvBlockBytes;
    } else {
        t.row0 = (i - s.run_count) * kChunk;
        t.from = 0, t.to = min(kChunk, s.single_count - t.row0);
        t.rec = nullptr, t.chunk = 0;
    }
    return t;
}
// The block's row at a place that has one.
__device__ __forceinline__ int kv_row(const KvRowsSmem &s, const KvTask &t, int p) {
    return t.run ? t.row0 + p - t.from : s.singles[t.row0 + p];
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, kAppendCtas<T>) kv_append_kernel(KvRowsArgs a) {
    __shared__ KvRowsSmem s;
    const int first = blockIdx.x * a.block_rows, head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    kv_rows_block(a, s, first);
    const int tasks = kv_tasks(s);
    uint32_t *turn = reinterpret_cast<uint32_t *>(s.turn[warp]);
    constexpr int kRow = kTurnRow / 4;
    for (int i = warp; i < tasks; i += kRowWarps) {
        const KvTask t = kv_task(s, i, head);
        Eight<T> x[2][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int p = 4 * j + (lane >> 3);
            const size_t at = first + kv_row(s, t, min(max(p, t.from), t.to - 1));
            x[0][j].load(static_cast<const T *>(a.k) + at * a.k_stride + head * kHeadDim + (lane & 7) * 8);
            x[1][j].load(static_cast<const T *>(a.v) + at * a.v_stride + head * kHeadDim + (lane & 7) * 8);
        }
#pragma unroll
        for (int which = 0; which < 2; which++) {
            float scale[4], inverse[4];
            row_scales(x[which], lane, scale, inverse);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int p = 4 * j + (lane >> 3);
                const uint2 w = quantize8(x[which][j], inverse[j]);
                turn[p * kRow + (lane & 7) * 2] = w.x, turn[p * kRow + (lane & 7) * 2 + 1] = w.y;
                if (p >= t.from && p < t.to && (lane & 7) == 0) {
                    const int row = kv_row(s, t, p), place = s.place[row];
                    uint8_t *rec = s.rec[row];
                    if (rec) {
                        rec += (size_t)head * kKvBlockBytes;
                        if (which) reinterpret_cast<float *>(rec + kVScaleOffset)[v_scale_index(place)] = scale[j];
                        else reinterpret_cast<float *>(rec + kKScaleOffset)[k_scale_index(place)] = scale[j];
                    }
                }
            }
            __syncwarp();
            if (t.run && which == 0) {
                // 16-byte chunk (32-dim step h, row & 7, column): words of positions r and r + 8, dims and dims + 16
                const int r = lane >> 2, c = lane & 3;
                const bool low = r >= t.from && r < t.to, high = r + 8 >= t.from && r + 8 < t.to;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t *dst = reinterpret_cast<uint32_t *>(t.rec + t.chunk * 1024 + h * 512 + lane * 16);
                    const uint32_t *src = turn + r * kRow + h * 8 + c;
                    const uint4 w = make_uint4(src[0], src[8 * kRow], src[4], src[8 * kRow + 4]);
                    if (low && high) {
                        *reinterpret_cast<uint4 *>(dst) = w;
                    } else {
                        if (low) dst[0] = w.x, dst[2] = w.z;
                        if (high) dst[1] = w.y, dst[3] = w.w;
                    }
                }
            } else if (t.run) {
                // lane -> positions 4 q .. of dims 4 c ..
                const int q = lane & 3;
                const bool all = 4 * q >= t.from && 4 * q + 4 <= t.to;
                if (4 * q + 4 > t.from && 4 * q < t.to) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int c = (lane >> 2) + 8 * h;
                        uint32_t b[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) b[j] = turn[(4 * q + j) * kRow + c];
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
            } else {
                // 16 lanes a single row, two rows an access (a row's key words lie in four sectors)
                const int c = lane & 15;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int p = 2 * j + (lane >> 4);
                    if (p >= t.to) break;
                    const int row = kv_row(s, t, p), place = s.place[row];
                    if (!s.rec[row]) continue;
                    uint8_t *rec = s.rec[row] + (size_t)head * kKvBlockBytes;
                    const uint32_t w = turn[p * kRow + c];
                    if (which == 0) *reinterpret_cast<uint32_t *>(rec + k_byte(place, 4 * c)) = w;
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++) rec[v_byte(place, 4 * c + e)] = (uint8_t)(w >> (8 * e));
                }
            }
        }
        __syncwarp();
    }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads, kGatherCtas<T>) kv_gather_kernel(KvRowsArgs a) {
    __shared__ KvRowsSmem s;
    const int first = blockIdx.x * a.block_rows, head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    kv_rows_block(a, s, first);
    const int tasks = kv_tasks(s);
    uint32_t *turn = reinterpret_cast<uint32_t *>(s.turn[warp]);
    constexpr int kRow = kTurnRow / 4;
    for (int i = warp; i < tasks; i += kRowWarps) {
        const KvTask t = kv_task(s, i, head);
        // scales of the places this lane's eights have
        float scale[2][4];
        uint4 key[2], dim[2];
        if (t.run) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                key[h] = __ldg(reinterpret_cast<const uint4 *>(t.rec + t.chunk * 1024 + h * 512 + lane * 16));
                dim[h] = __ldg(reinterpret_cast<const uint4 *>(t.rec + v_byte(t.chunk * kChunk, lane + 32 * h)));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int p = 4 * j + (lane >> 3);
            scale[0][j] = scale[1][j] = 0.0f;
            if (p >= t.from && p < t.to) {
                const int row = kv_row(s, t, p), place = s.place[row];
                const uint8_t *rec = s.rec[row];
                if (rec) {
                    rec += (size_t)head * kKvBlockBytes;
                    scale[0][j] = __ldg(reinterpret_cast<const float *>(rec + kKScaleOffset) + k_scale_index(place));
                    scale[1][j] = __ldg(reinterpret_cast<const float *>(rec + kVScaleOffset) + v_scale_index(place));
                } else if (s.bad[row]) {  // NaN; a padding row gives zeros
                    scale[0][j] = scale[1][j] = __int_as_float(0x7fc00000);
                }
            }
        }
#pragma unroll
        for (int which = 0; which < 2; which++) {
            __syncwarp();
            if (t.run && which == 0) {
                const int r = lane >> 2, c = lane & 3;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t *dst = turn + r * kRow + h * 8 + c;
                    dst[0] = key[h].x, dst[8 * kRow] = key[h].y, dst[4] = key[h].z, dst[8 * kRow + 4] = key[h].w;
                }
            } else if (t.run) {
                // dims as rows of 16 bytes, turned around to positions as rows
#pragma unroll
                for (int h = 0; h < 2; h++) *reinterpret_cast<uint4 *>(turn + (lane + 32 * h) * 4) = dim[h];
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
                    for (int j = 0; j < 4; j++) turn[(4 * q + j) * kRow + (lane >> 2) + 8 * h] = b[h][j];
            } else {
                // 16 lanes a single row, two rows an access (a row's key words lie in four sectors)
                const int c = lane & 15;
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int p = 2 * j + (lane >> 4);
                    const int row = p < t.to ? kv_row(s, t, p) : 0, place = s.place[row];
                    w[j] = 0;
                    if (p >= t.to || !s.rec[row]) continue;
                    const uint8_t *rec = s.rec[row] + (size_t)head * kKvBlockBytes;
                    if (which == 0) w[j] = __ldg(reinterpret_cast<const uint32_t *>(rec + k_byte(place, 4 * c)));
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++) w[j] |= (uint32_t)__ldg(rec + v_byte(place, 4 * c + e)) << (8 * e);
                }
#pragma unroll
                for (int j = 0; j < 8; j++) turn[(2 * j + (lane >> 4)) * kRow + c] = w[j];
            }
            __syncwarp();
            T *out = static_cast<T *>(which ? a.v_out : a.k_out);
            const long long stride = which ? a.v_stride : a.k_stride;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int p = 4 * j + (lane >> 3);
                if (p < t.from || p >= t.to) continue;
                const uint2 w = make_uint2(turn[p * kRow + (lane & 7) * 2], turn[p * kRow + (lane & 7) * 2 + 1]);
                Eight<T> x;
                scale8(w, scale[which][j], x);
                x.store(out + (size_t)(first + kv_row(s, t, p)) * stride + head * kHeadDim + (lane & 7) * 8);
            }
        }
        __syncwarp();
    }
}

// Rows a block, whose CTAs (one a head) are small because single rows cost an SM's load/store unit a clock a byte of
// values: 32 where that leaves every SM two blocks, else 16, a warp's share of single rows.  (8 heads, bf16, append and
// gather with 32 and with 16: 16384 rows of runs 32 + 21 and 40 + 27 us, 4096 8 + 6 and 12 + 9, 1243 single rows
// 14 + 10 and 13 + 9.)
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
