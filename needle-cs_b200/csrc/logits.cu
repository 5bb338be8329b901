// Penalties, biases and masks on logits, before a sampler reads them.
//
// Per row and vocabulary id, in this order (each step one IEEE operation):
//   repetition: an id anywhere in the row's tokens: x > 0 ? x / r : x * r
//   frequency, presence: an id that occurs n > 0 times among the row's output
//     tokens (those behind its prompt): x - f * n, then - p
//   bias: the row's last entry for the id is added
//   mask: an id whose bit is clear becomes -inf, whatever it was
// A CTA takes one row's slice of the vocabulary: the occurrences of the slice's
// ids are counted in shared memory (integers, so their order does not matter)
// from the row's tokens, then the slice streams through once.
#include "common.cuh"

namespace ndl {

constexpr int kLogitSlice = 4096;   // ids per CTA: 32 KB of counts and bias entries
constexpr int kLogitThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;  // in the row's tokens; the low bits count its output tokens

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

__global__ void __launch_bounds__(kLogitThreads) logits_process_kernel(LogitsArgs a) {
    __shared__ uint32_t count[kLogitSlice];
    __shared__ int32_t bias[kLogitSlice];
    const int row = blockIdx.y, first = blockIdx.x * kLogitSlice;
    const int n = min(kLogitSlice, a.vocab - first);
    for (int i = threadIdx.x; i < n; i += kLogitThreads) count[i] = 0, bias[i] = -1;
    __syncthreads();
    if (a.token_offsets && a.n_tokens > 0) {
        const int begin = max(0, a.token_offsets[row]), end = min(a.n_tokens, a.token_offsets[row + 1]);
        const int output = a.prompt_lens ? max(0, a.prompt_lens[row]) : 0;  // tokens from here on are the output
        for (int i = begin + threadIdx.x; i < end; i += kLogitThreads) {
            const int id = a.tokens[i] - first;
            if ((unsigned)id >= (unsigned)n) continue;
            atomicOr(&count[id], kSeen);
            if (i - begin >= output) atomicAdd(&count[id], 1u);
        }
    }
    if (a.bias_offsets && a.n_bias > 0) {
        const int begin = max(0, a.bias_offsets[row]), end = min(a.n_bias, a.bias_offsets[row + 1]);
        for (int i = begin + threadIdx.x; i < end; i += kLogitThreads) {
            const int id = a.bias_ids[i] - first;
            if ((unsigned)id < (unsigned)n) atomicMax(&bias[id], i);
        }
    }
    __syncthreads();
    const float r = a.repetition ? a.repetition[row] : 1.0f;
    const float f = a.frequency ? a.frequency[row] : 0.0f;
    const float p = a.presence ? a.presence[row] : 0.0f;
    int mrow = -1;
    if (a.mask) {
        mrow = a.mask_index ? a.mask_index[row] : row;
        if (mrow >= a.mask_rows) {
            if (threadIdx.x == 0 && a.status) atomicOr(a.status, 2);
        }
    }
    const bool bad_mask = a.mask && mrow >= a.mask_rows;
    const uint32_t *mask = mrow >= 0 && !bad_mask ? a.mask + (size_t)mrow * a.words : nullptr;
    for (int i = threadIdx.x; i < n; i += kLogitThreads) {
        const int id = first + i;
        float x = a.x[(size_t)row * a.ldx + id];
        const uint32_t c = count[i];
        if (c) {
            if (a.repetition) x = x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
            const uint32_t times = c & ~kSeen;
            if (times) {
                if (a.frequency) x = __fsub_rn(x, __fmul_rn(f, (float)times));
                if (a.presence) x = __fsub_rn(x, p);
            }
        }
        if (bias[i] >= 0) x = __fadd_rn(x, a.bias_values[bias[i]]);
        if (mask && !(id < 32 * a.words && ((mask[id >> 5] >> (id & 31)) & 1u))) x = -INFINITY;
        if (bad_mask) x = __int_as_float(0x7fc00000);
        a.y[(size_t)row * a.ldy + id] = x;
    }
}

}  // namespace ndl

using namespace ndl;

extern "C" NDL_API int ndl_logits_process(const float *x, long long ldx, float *y, long long ldy, int rows, int vocab,
                                          const int32_t *tokens, int n_tokens, const int32_t *token_offsets,
                                          const int32_t *prompt_lens, const float *repetition, const float *frequency,
                                          const float *presence, const int32_t *bias_ids, const float *bias_values,
                                          int n_bias, const int32_t *bias_offsets, const uint32_t *mask, int mask_rows,
                                          int words, const int32_t *mask_index, int *status, void *stream) {
    NDL_REQUIRE(rows >= 0 && vocab >= 1 && n_tokens >= 0 && n_bias >= 0, "bad logits geometry");
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
    const dim3 grid((vocab + kLogitSlice - 1) / kLogitSlice, rows);
    logits_process_kernel<<<grid, kLogitThreads, 0, (cudaStream_t)stream>>>(a);
    return check_launch("logits_process");
}
