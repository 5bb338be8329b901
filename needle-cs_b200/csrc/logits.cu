// Penalties, biases and masks on logits, before a sampler reads them.
//
// Per row and vocabulary id, in this order (each step one IEEE operation):
//   repetition: an id anywhere in the row's tokens: x > 0 ? x / r : x * r
//   frequency, presence: an id that occurs n > 0 times among the row's output
//     tokens (those behind its prompt): x - f * n, then - p
//   bias: the row's last entry for the id is added
//   mask: an id whose bit is clear becomes -inf, whatever it was
// Bound by memory: 8 bytes an id.  A small call is one kernel: a CTA takes one
// row's slice of the vocabulary, counts the occurrences of the slice's ids in
// shared memory (integers, so their order does not matter) from the row's
// tokens, then streams the slice through, four ids a thread and access.  With
// many ids the counting's dependent reads leave memory idle: there a kernel
// streams rows and masks, and a second, launched early, gathers the lists' ids
// meanwhile and then goes over those alone.  Rows of 51865 ids with lists of up
// to 1024 tokens, one kernel against two: 40 rows 8.2 and 10.0 us, 64 rows 11.0
// and 11.1, 128 rows 16.2 and 14.0, 256 rows 34.6 and 24.8 (29 with inputs that
// the cache does not hold: 3.6 TB/s).  One row is the launch and one trip to
// memory after another (offsets, tokens, counts): 5 us.
//
// A slice counts its places from the 16-byte boundary at or before the row's
// start, so accesses are aligned whatever the row stride is.
#include "common.cuh"

namespace ndl {

constexpr int kLogitThreads = 256, kLogitPer = 16;      // ids a thread: four accesses of four
constexpr int kLogitSlice = kLogitThreads * kLogitPer;  // ids a CTA: 32 KB of counts and bias entries
constexpr uint32_t kSeen = 0x80000000u;                 // in the row's prompt; the low bits count its output tokens
constexpr long long kManyIds = 3 << 20;                 // from here on in two kernels: there both take as long (above)

struct LogitsArgs {
    const float *x;
    float *y;
    long long ldx, ldy;
    int rows, vocab;
    const int32_t *tokens, *token_offsets, *prompt_lens;
    int n_tokens;
    const float *repetition, *frequency, *presence;
    const int32_t *bias_ids, *bias_offsets;
    const float *bias_values;
    int n_bias;
    const uint32_t *mask;
    int mask_rows, words;
    const int32_t *mask_index;
    int *status;
};

// A CTA's slice of a row: places 0 .. n - 1 hold ids first .. (those before id 0 hold nothing).
struct LogitsSlice {
    int row, first, n;
    const float *x;  // of place 0
    float *y;
    const uint32_t *mask;  // the row's, null: none
    bool bad;              // the row's mask does not exist
    template <bool kVec>
    __device__ __forceinline__ static LogitsSlice of(const LogitsArgs &a, int row, int slice) {
        LogitsSlice s;
        s.row = row;
        const float *x = a.x + (size_t)s.row * a.ldx;
        const int shift = kVec ? (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3) : 0;
        s.first = slice * kLogitSlice - shift;
        s.n = min(kLogitSlice, a.vocab - s.first);
        s.x = x + s.first, s.y = a.y + (size_t)s.row * a.ldy + s.first;
        int mrow = -1;
        if (a.mask) mrow = a.mask_index ? a.mask_index[s.row] : s.row;
        s.bad = a.mask && mrow >= a.mask_rows;
        s.mask = mrow >= 0 && !s.bad ? a.mask + (size_t)mrow * a.words : nullptr;
        return s;
    }
    __device__ __forceinline__ bool holds(int place) const { return place < n && first + place >= 0; }
    // four places from `place` on
    template <bool kVec>
    __device__ __forceinline__ bool whole(int place) const {
        return kVec && place + 4 <= n && first + place >= 0;
    }
    template <bool kVec>
    __device__ __forceinline__ void load(int place, float *v) const {
        if (whole<kVec>(place)) {
            const float4 q = *reinterpret_cast<const float4 *>(x + place);
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = holds(place + e) ? x[place + e] : 0.0f;
        }
    }
    template <bool kVec>
    __device__ __forceinline__ void store(int place, const float *v) const {
        if (whole<kVec>(place)) {
            *reinterpret_cast<float4 *>(y + place) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (holds(place + e)) y[place + e] = v[e];
        }
    }
    // Bits of four ids: the first one's word, and the next where they reach into it.
    __device__ __forceinline__ uint32_t bits(const LogitsArgs &a, int place) const {
        if (!mask) return 0xF;
        const int id = first + place, word = id >> 5;  // (-1 before the row)
        const uint32_t lo = word >= 0 && word < a.words ? __ldg(mask + word) : 0;
        const uint32_t hi = (id & 31) > 28 && word + 1 < a.words ? __ldg(mask + word + 1) : 0;
        return __funnelshift_r(lo, hi, id & 31);
    }
    __device__ __forceinline__ float masked(float v, uint32_t bits, int e) const {
        if (!(bits >> e & 1)) v = -INFINITY;
        return bad ? __int_as_float(0x7fc00000) : v;
    }
};

// The slice's counts and last bias entries, from the row's lists.
struct LogitsCounts {
    uint32_t count[kLogitSlice];
    int32_t bias[kLogitSlice];
};
struct LogitsLists {
    int t0, t1, b0, b1;  // the row's tokens and biases
    float r, f, p;
    __device__ __forceinline__ explicit LogitsLists(const LogitsArgs &a, int row) : t0(0), t1(0), b0(0), b1(0) {
        if (a.token_offsets && a.n_tokens > 0) t0 = max(0, a.token_offsets[row]), t1 = min(a.n_tokens, a.token_offsets[row + 1]);
        if (a.bias_offsets && a.n_bias > 0) b0 = max(0, a.bias_offsets[row]), b1 = min(a.n_bias, a.bias_offsets[row + 1]);
        r = a.repetition ? a.repetition[row] : 1.0f;
        f = a.frequency ? a.frequency[row] : 0.0f;
        p = a.presence ? a.presence[row] : 0.0f;
    }
    __device__ __forceinline__ bool any() const { return t0 < t1 || b0 < b1; }
    // Place of a list's id in the slice, or -1.
    __device__ __forceinline__ static int place(const LogitsSlice &s, int id) {
        const unsigned at = (unsigned)id - (unsigned)s.first;
        return id >= 0 && s.n > 0 && at < (unsigned)s.n ? (int)at : -1;
    }
    __device__ __forceinline__ void tally(const LogitsArgs &a, const LogitsSlice &s, LogitsCounts &c) const {
        for (int i = threadIdx.x * 4; i < kLogitSlice; i += blockDim.x * 4) {
            *reinterpret_cast<uint4 *>(c.count + i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<int4 *>(c.bias + i) = make_int4(-1, -1, -1, -1);
        }
        const int prompt = a.prompt_lens ? max(0, a.prompt_lens[s.row]) : 0;  // tokens from here on are the output
        __syncthreads();
        for (int i = t0 + threadIdx.x; i < t1; i += blockDim.x) {
            const int at = place(s, a.tokens[i]);
            if (at < 0) continue;
            // the prompt's tokens set the id's bit, the output's count
            if (i - t0 >= prompt) atomicAdd(&c.count[at], 1u);
            else atomicOr(&c.count[at], kSeen);
        }
        for (int i = b0 + threadIdx.x; i < b1; i += blockDim.x) {
            const int at = place(s, a.bias_ids[i]);
            if (at >= 0) atomicMax(&c.bias[at], i);
        }
        __syncthreads();
    }
    __device__ __forceinline__ float apply(const LogitsArgs &a, float v, uint32_t count, int bias) const {
        if (count) {
            if (a.repetition) v = v > 0.0f ? __fdiv_rn(v, r) : __fmul_rn(v, r);
            const uint32_t times = count & ~kSeen;
            if (times) {
                if (a.frequency) v = __fsub_rn(v, __fmul_rn(f, (float)times));
                if (a.presence) v = __fsub_rn(v, p);
            }
        }
        return bias >= 0 ? __fadd_rn(v, a.bias_values[bias]) : v;
    }
};

// All at once.  kVec: the rows of both matrices lie alike to 16-byte boundaries.
template <bool kVec>
__global__ void __launch_bounds__(kLogitThreads) logits_process_kernel(LogitsArgs a) {
    __shared__ __align__(16) LogitsCounts c;
    const LogitsSlice s = LogitsSlice::of<kVec>(a, blockIdx.y, blockIdx.x);
    float x[kLogitPer];
#pragma unroll
    for (int j = 0; j < kLogitPer; j += 4) s.load<kVec>(j * kLogitThreads + threadIdx.x * 4, x + j);
    const LogitsLists l(a, s.row);
    if (s.bad && threadIdx.x == 0 && blockIdx.x == 0 && a.status) atomicOr(a.status, 2);
    if (l.any()) l.tally(a, s, c);
#pragma unroll
    for (int j = 0; j < kLogitPer; j += 4) {
        const int i = j * kLogitThreads + threadIdx.x * 4;
        if (i >= s.n) break;
        const uint32_t bits = s.bits(a, i);
        uint4 n = make_uint4(0, 0, 0, 0);
        int4 b = make_int4(-1, -1, -1, -1);
        if (l.any()) n = *reinterpret_cast<const uint4 *>(c.count + i), b = *reinterpret_cast<const int4 *>(c.bias + i);
        const uint32_t ns[4] = {n.x, n.y, n.z, n.w};
        const int bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; e++) x[j + e] = s.masked(l.apply(a, x[j + e], ns[e], bs[e]), bits, e);
        s.store<kVec>(i, x + j);
    }
}

// Rows and masks alone.
template <bool kVec>
__global__ void __launch_bounds__(kLogitThreads) logits_stream_kernel(LogitsArgs a) {
    pdl_trigger();
    const LogitsSlice s = LogitsSlice::of<kVec>(a, blockIdx.y, blockIdx.x);
    if (s.bad && threadIdx.x == 0 && blockIdx.x == 0 && a.status) atomicOr(a.status, 2);
    float x[kLogitPer];
    uint32_t bits[kLogitPer / 4];
#pragma unroll
    for (int j = 0; j < kLogitPer; j += 4) {
        const int i = j * kLogitThreads + threadIdx.x * 4;
        s.load<kVec>(i, x + j);
        bits[j / 4] = s.bits(a, i);
    }
#pragma unroll
    for (int j = 0; j < kLogitPer; j += 4) {
#pragma unroll
        for (int e = 0; e < 4; e++) x[j + e] = s.masked(x[j + e], bits[j / 4], e);
        s.store<kVec>(j * kLogitThreads + threadIdx.x * 4, x + j);
    }
}

// The ids of a row's lists, over the streamed row (whose masked places keep their -inf): a CTA a row gathers them in a
// hash table in shared memory (counts and last bias entries again, so the order of insertion does not matter).  Lists
// that are too long for it go slice by slice.
constexpr int kListThreads = 512, kTableSlots = 8192, kTableEntries = kTableSlots / 2;
constexpr size_t kTableBytes = (size_t)kTableSlots * 3 * 4;
static_assert(sizeof(LogitsCounts) <= kTableBytes, "a slice's counts fit the table's place");

__global__ void __launch_bounds__(kListThreads) logits_lists_kernel(LogitsArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int row = blockIdx.x;
    const LogitsLists l(a, row);
    LogitsSlice s = LogitsSlice::of<false>(a, row, 0);
    if (s.bad || !l.any()) {
        pdl_wait();  // what follows this kernel on the stream may go by its end alone
        return;
    }
    const auto fix = [&](int at, uint32_t count, int bias) {
        if (s.bits(a, at) & 1) s.y[at] = l.apply(a, s.x[at], count, bias);
    };
    const int entries = (l.t1 > l.t0 ? l.t1 - l.t0 : 0) + (l.b1 > l.b0 ? l.b1 - l.b0 : 0);
    if (entries <= kTableEntries) {
        int slots = 64;
        while (slots < 2 * entries) slots *= 2;
        int32_t *key = reinterpret_cast<int32_t *>(smem), *bias = key + slots;
        uint32_t *count = reinterpret_cast<uint32_t *>(bias + slots);
        for (int i = threadIdx.x; i < slots; i += kListThreads) key[i] = -1, bias[i] = -1, count[i] = 0;
        const int prompt = a.prompt_lens ? max(0, a.prompt_lens[row]) : 0;  // tokens from here on are the output
        __syncthreads();
        const auto slot_of = [&](int id) {  // half of the slots stay free: the walk ends
            int i = (int)(((uint32_t)id * 2654435769u) >> 7) & (slots - 1);
            for (;; i = (i + 1) & (slots - 1)) {
                const int old = atomicCAS(&key[i], -1, id);
                if (old == -1 || old == id) return i;
            }
        };
        for (int i = l.t0 + threadIdx.x; i < l.t1; i += kListThreads) {
            const int id = a.tokens[i];
            if (id < 0 || id >= a.vocab) continue;
            uint32_t *n = &count[slot_of(id)];
            // the prompt's tokens set the id's bit, the output's count
            if (i - l.t0 >= prompt) atomicAdd(n, 1u);
            else atomicOr(n, kSeen);
        }
        for (int i = l.b0 + threadIdx.x; i < l.b1; i += kListThreads) {
            const int id = a.bias_ids[i];
            if (id >= 0 && id < a.vocab) atomicMax(&bias[slot_of(id)], i);
        }
        __syncthreads();
        pdl_wait();  // the stream's end
        for (int i = threadIdx.x; i < slots; i += kListThreads)
            if (key[i] >= 0) fix(key[i], count[i], bias[i]);
        return;
    }
    LogitsCounts &c = *reinterpret_cast<LogitsCounts *>(smem);
    pdl_wait();
    const int slices = (a.vocab + kLogitSlice - 1) / kLogitSlice;
    for (int k = 0; k < slices; k++) {
        s = LogitsSlice::of<false>(a, row, k);
        __syncthreads();
        l.tally(a, s, c);
        for (int i = threadIdx.x; i < s.n; i += kListThreads)
            if (c.count[i] || c.bias[i] >= 0) fix(i, c.count[i], c.bias[i]);
    }
}

template <bool kVec>
static int launch_logits(const LogitsArgs &a, cudaStream_t stream) {
    const dim3 grid((unsigned)(((long long)a.vocab + (kVec ? 3 : 0) + kLogitSlice - 1) / kLogitSlice), a.rows);
    if ((long long)a.rows * a.vocab < kManyIds) {
        logits_process_kernel<kVec><<<grid, kLogitThreads, 0, stream>>>(a);
        return check_launch("logits_process");
    }
    logits_stream_kernel<kVec><<<grid, kLogitThreads, 0, stream>>>(a);
    const int rc = check_launch("logits_stream");
    if (rc != NDL_OK || (!a.n_tokens && !a.n_bias)) return rc;
    static DeviceOnce attribute;  // the attribute belongs to the kernel on one device
    const int st = attribute.run([] {
        const cudaError_t e = cudaFuncSetAttribute(logits_lists_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kTableBytes);
        return e == cudaSuccess ? (int)NDL_OK : set_error(NDL_ERR_CUDA, "logits smem: %s", cudaGetErrorString(e));
    });
    if (st != NDL_OK) return st;
    PdlScope early(true);  // the lists' launch overlaps the stream; it waits for its end before writing
    launch_kernel(logits_lists_kernel, dim3(a.rows), dim3(kListThreads), kTableBytes, stream, a);
    return check_launch("logits_lists");
}

}  // namespace ndl

using namespace ndl;

extern "C" NDL_API int ndl_logits_process(const float *x, long long ldx, float *y, long long ldy, int rows, int vocab,
                                          const int32_t *tokens, int n_tokens, const int32_t *token_offsets,
                                          const int32_t *prompt_lens, const float *repetition, const float *frequency,
                                          const float *presence, const int32_t *bias_ids, const float *bias_values,
                                          int n_bias, const int32_t *bias_offsets, const uint32_t *mask, int mask_rows,
                                          int words, const int32_t *mask_index, int *status, void *stream) {
    NDL_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= 1 << 30 && n_tokens >= 0 && n_bias >= 0, "bad logits geometry");
    if (rows == 0) return NDL_OK;
    NDL_REQUIRE(x && y, "null pointer");
    NDL_REQUIRE(ldx >= vocab && ldy >= vocab, "row strides %lld, %lld below the vocabulary of %d", ldx, ldy, vocab);
    NDL_REQUIRE(rows <= 65535, "%d rows; at most 65535", rows);
    NDL_REQUIRE(x != y || ldx == ldy, "in place with two row strides");
    // an empty list may come as a null pointer: the offsets say whether there are lists at all
    NDL_REQUIRE(token_offsets || !(tokens || repetition || frequency || presence || prompt_lens),
                "tokens and penalties need token offsets");
    NDL_REQUIRE(tokens || n_tokens == 0, "%d tokens: null pointer", n_tokens);
    NDL_REQUIRE(bias_offsets || !(bias_ids || bias_values), "biases need offsets");
    NDL_REQUIRE((bias_ids && bias_values) || n_bias == 0, "%d biases: null pointer", n_bias);
    NDL_REQUIRE(!mask || (words >= 1 && mask_rows >= 1), "mask of %d rows of %d words", mask_rows, words);
    NDL_REQUIRE(!mask || mask_index || mask_rows >= rows, "%d mask rows for %d rows", mask_rows, rows);
    NDL_REQUIRE(mask || !mask_index, "mask index without masks");
    LogitsArgs a{x, y, ldx, ldy, rows, vocab, tokens, token_offsets, prompt_lens, n_tokens, repetition, frequency,
                 presence, bias_ids, bias_offsets, bias_values, n_bias, mask, mask_rows, words, mask_index, status};
    NDL_REQUIRE(aligned(x, 4) && aligned(y, 4), "misaligned pointer");
    const bool vec = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) & 15) == 0 && (ldx - ldy) % 4 == 0;
    return vec ? launch_logits<true>(a, (cudaStream_t)stream) : launch_logits<false>(a, (cudaStream_t)stream);
}
