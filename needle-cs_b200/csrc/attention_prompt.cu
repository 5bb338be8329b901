// Whole-prompt attention over the paged int8 cache, on the fifth-generation
// tensor cores.
//
// A CTA takes up to 384 packed rows (three tiles of 128; fp32: two) of one
// sequence and kv head; packed row m is query m / group of the sequence and
// query head m % group of the kv head's group, so a page of keys and values
// serves every query head that shares it.  It walks the pages its rows see, one
// (64 positions) a step, with the softmax's running maximum and sum:
//   S = Q K^T       tcgen05.mma, fp16 operands, fp32 accumulator in TMEM
//   e = 2^(f S - m),  l += e,  P = e,  O += P V
// Every operand is brought into fp16's range by a power of two: a query row's
// largest element to [2^10, 2^11) (16-bit queries stay exact), the key scales of
// a step to below 2^8 (f undoes both), the value scales to below 2^8 by that of
// the largest so far (O is rescaled where it grows).  m follows the true maximum
// only where that is 7 binary orders above it, so O is rescaled on few steps.
// What an operand rounds to:
//   bf16  keys, values (code * scale) and P one fp16 each: 2^-11 a term, an
//         eighth of the result's own rounding;
//   fp16  keys and values as bare codes (exact), their scales on S and on P,
//         which rounds as the result does;
//   fp32  as fp16, and queries and P in two parts: 2^-21 throughout.
// A scale a column costs the softmax threads (thread = row) a shared-memory
// wavefront a column and warp, so for bf16 both go into the operands (8192 rows
// of 32 heads over 8: 730 us against 967 with both on S and P, at the time).
// Keys in two parts would keep one of the scales out of fp16's and fp32's
// softmax at 4 and 8 more products a step: fp16 6 % faster over long prompts,
// fp32 5 % slower.
//
// Warps: 4 softmax warps a tile (maximum and sum need no exchange), 4 that
// convert pages (int8 records -> fp16 tiles in shared memory, 128-byte swizzled
// rows), 1 that copies the records, 1 a tile that issues its MMAs.  P goes back
// to TMEM, from where the second product takes it as its A operand.
//
// Bound by the softmax warps: a column costs a row an exponential (16 a clock
// and SM) and some six instructions more.  8192 rows of 32 heads over 8, bf16,
// causal: 461 us (0.60 PFLOP/s), where the two products alone would take 163 at
// the library's rate; of 478 it took 434 without the exponentials and 473 without
// the conversions.  The three tiles hide one another's waits: two took 524, two
// with steps of 128 columns 545, one tile and two CTAs an SM 664.  Short prompts
// are bound by what a CTA does around its steps (a step of three tiles takes 1.4
// to 1.7 us, of fp32's two 1.8, all else 9 to 11) and by the CTAs that come last:
// 32 prompts of up to 384 rows, 8 heads, fp32: 41 us; one of 37 rows: 8 us.
// (Two threads a row of fp32, each with half the columns and an output of its
// own, took as long a step and 1 us more around them.)
//
// A value scale that is no number would reach rows that do not see its
// position through the product (0 * NaN): it is replaced by 0 and its key
// scale by NaN, which only the rows that see the position take up.
#include <float.h>

#include "attention_math.cuh"
#include "tc.cuh"

namespace ndl {

namespace {

constexpr int kTileRows = 128;  // MMA rows: TMEM lanes
constexpr int kTileBytes = kTileRows * kHeadDim * 2;      // 16 KB of queries
constexpr int kPageTile = kPagePositions * kHeadDim * 2;  // 8 KB of keys or values
constexpr uint32_t kPromptWait = 1u << 22;                // waits of about a microsecond: a few seconds
constexpr int kTmemCols = 512;
constexpr int kConvertWarps = 4;

// The forms of the element types (above).
template <class T>
struct Step {
    static constexpr bool kSplit = sizeof(T) == 4;                       // queries and P in two parts
    static constexpr bool kFold = __is_same(T, __nv_bfloat16);           // scales on keys and values, else on S and P
    static constexpr int kQParts = kSplit ? 2 : 1;
    // Tiles of 128 rows: three (above); the softmax of fp32, with a second part of each probability, needs the
    // registers of two.
    static constexpr int kTiles = kSplit ? 2 : 3, kRows = kTiles * kTileRows;
    // Pages a step: one; with two the scores' registers spill or leave room for two tiles alone (above).
    static constexpr int kPages = 1, kCols = kPages * kPagePositions;
    static constexpr int kStages = 4;  // converted steps in flight
    static constexpr int kRaw = 3;     // steps of records as they lie in the pages
    // TMEM columns: scores, outputs, probabilities (two fp16 a column; fp32: then their second parts) of the tiles
    static constexpr int kS = 0, kO = kTiles * kCols, kP = kO + kTiles * kHeadDim, kPCols = kCols / 2;
    static constexpr int kLo = kTiles * kPCols;
    // fp32: the accumulators truncate what is added, a bias that grows with the steps; so every kFlush steps O goes over
    // to a sum, which rounds (a prompt of 1408 rows is off by 1.4e-6 without, 0.9e-6 with 8 steps, 0.6e-6 with 4; a
    // time costs 1 us: a step takes 1.6 us without, 1.8 with 8 steps).
    static constexpr int kFlush = kSplit ? 8 : 1, kSum = kLo + kP + kTiles * kPCols;
    static_assert((kSplit ? kSum + kTiles * kHeadDim : kP + kTiles * kPCols) <= kTmemCols, "TMEM columns");
    // Warps: softmax, converters, then a group of one MMA warp a tile and one that copies.
    static constexpr int kConvertWarp = 4 * kTiles, kMmaWarp = kConvertWarp + kConvertWarps, kCopyWarp = kMmaWarp + 3;
    static constexpr int kThreads = 32 * (kMmaWarp + 4);
    // 16-byte chunks of a query row, and the row (of a warp's 32) whose chunk lane % kRowChunks access i takes.
    static constexpr int kRowChunks = kHeadDim * (int)sizeof(T) / 16;
    __device__ static constexpr int chunk_row(int i, int lane) { return i * (32 / kRowChunks) + lane / kRowChunks; }
    // Registers a thread: what the launch gives each (128 or 96), shared out anew: the softmax warps hold a row's scores.
    static constexpr int kLaunchRegs = kTiles == 2 ? 128 : 96;
    static constexpr int kSoftmaxRegs = kTiles == 2 ? 184 : 128, kConvertRegs = kTiles == 2 ? 96 : 64;
    static constexpr int kMmaRegs = kTiles == 2 ? 48 : 32;
    static_assert(kTiles * kSoftmaxRegs + kConvertRegs + kMmaRegs == (kTiles + 2) * kLaunchRegs, "the launch's registers");
};

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
struct PromptSmem {
    using St = Step<T>;
    uint8_t q[St::kTiles][St::kQParts][kTileBytes];  // 1024-byte aligned
    uint8_t k[St::kStages][St::kPages][kPageTile], v[St::kStages][St::kPages][kPageTile];
    uint8_t raw[St::kRaw][St::kPages][kKvBlockBytes];
    float scales[kConvertWarps][2][St::kPages][kPagePositions];  // each converter warp's copy: keys, values
    __align__(16) float ks[St::kStages][St::kFold ? 4 : St::kCols], vs[St::kStages][St::kFold ? 4 : St::kCols];
    float key_factor[St::kStages];  // 2^(the keys' exponent), the scale of their scores
    int exponent[St::kStages];      // of the value scales so far
    uint64_t raw_full[St::kRaw], kv_full[St::kStages], kv_empty[St::kStages];
    int missing[St::kRaw];  // bit g: the step's page g is not in the pool
    uint64_t s_full[St::kTiles], s_free[St::kTiles], p_full[St::kTiles], pv_done[St::kTiles];
    uint64_t q_full, drained[St::kTiles];
    uint32_t tmem;
    // this CTA's work: a sequence (rows 0: none) and the kRows-row tile of it
    int first_row, rows, slot, pos, tile;
    volatile int abort;
};

// Where 16-byte chunk j of a tile's row lies before it is normalised and after it is attended: in the swizzled rows of
// the query tiles (fp32: the second eight chunks in the second part's).
template <class T>
__device__ __forceinline__ uint8_t *row_chunk(PromptSmem<T> &s, int tile, int row, int j) {
    return &s.q[tile][j >> 3][row * 128 + (((j & 7) ^ (row & 7)) << 4)];
}
// 16 bytes to shared memory, zeros unless they are `there` (the address is valid all the same).
__device__ __forceinline__ void async_chunk(void *dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0)
                 : "memory");
}

// kind::f16, fp32 accumulator, A and B fp16, both K-major.
constexpr uint32_t idesc_f16(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Warp-converged: every lane calls, one elected lane issues.
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
            r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr));
}
// Bounded wait of a whole warp: a plain test first (the phase is mostly complete already), then suspending ones.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort) {
    if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    const bool ok = mbar_wait_bounded(bar, parity, kPromptWait);
    return __all_sync(0xffffffffu, ok && !*abort);
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <class T>
__global__ void __launch_bounds__(Step<T>::kThreads, 1) attention_prompt_kernel(PromptArgs a) {
    using St = Step<T>;
    constexpr bool kSplit = St::kSplit;
    constexpr int kStages = St::kStages, kPages = St::kPages, kCols = St::kCols, kTiles = St::kTiles;
    constexpr int kCtaRows = St::kRows, kMmaWarp = St::kMmaWarp;
    extern __shared__ uint8_t smem_raw[];
    PromptSmem<T> &s =
        *reinterpret_cast<PromptSmem<T> *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_head = blockIdx.x % a.c.heads, work = blockIdx.x / a.c.heads;
    const int group = a.heads / a.c.heads;

    // This CTA's tile: sequences hold ceil(rows * group / kCtaRows) tiles each.
    if (warp == 0) {
        bool found = false;
        if (lane == 0) s.first_row = s.rows = s.slot = s.pos = s.tile = 0, s.abort = 0;
        __syncwarp();  // before the lane that finds the work
        int before = 0;
        for (int base = 0; base < a.sequences && !found; base += 32) {
            const int i = base + lane;
            int first = 0, n = 0, slot = 0, pos = 0, tiles = 0;
            if (i < a.sequences) {
                const int b = a.seq_rows[i], e = a.seq_rows[i + 1];
                slot = a.seq_slot[i], pos = a.seq_pos[i];
                if (b >= 0 && e >= b && e <= a.rows) {
                    first = b, n = e - b;
                    tiles = (int)(((long long)n * group + kCtaRows - 1) / kCtaRows);
                }
            }
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const int at = work - (before + sum - tiles);
            const bool mine = at >= 0 && at < tiles;
            if (mine) {  // the last tile, which sees the most pages, first
                s.first_row = first, s.rows = n, s.slot = slot, s.pos = pos, s.tile = tiles - 1 - at;
            }
            found = __any_sync(0xffffffffu, mine);
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (blockIdx.x == 0)
            for (int i = lane; i < a.sequences; i += 32) {
                const int b = a.seq_rows[i], e = a.seq_rows[i + 1];
                if ((b < 0 || e < b || e > a.rows) && a.c.status) atomicOr(a.c.status, kStatusBadPage);
            }
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            mbar_init(&s.q_full, 4 * kTiles);
            for (int t = 0; t < kTiles; t++) mbar_init(&s.drained[t], 1);
            for (int i = 0; i < St::kRaw; i++) mbar_init(&s.raw_full[i], 1);
            for (int i = 0; i < kStages; i++) mbar_init(&s.kv_full[i], kConvertWarps), mbar_init(&s.kv_empty[i], kTiles);
            for (int t = 0; t < kTiles; t++)
                mbar_init(&s.s_full[t], 2), mbar_init(&s.s_free[t], 4), mbar_init(&s.p_full[t], 4),
                    mbar_init(&s.pv_done[t], 1);
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s.tmem, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s.tmem;
    const int n = s.rows, first_row = s.first_row, slot = s.slot, start = s.pos;
    const bool ok_seq = slot >= 0 && slot < a.c.slots && start >= 0 &&
                        (long long)start + n <= (long long)a.c.max_pages * kPagePositions;
    // (rows x heads is below 2^31)
    const unsigned packed = (unsigned)n * group, m0 = (unsigned)s.tile * kCtaRows;
    // the pages its rows see, from page0 on in steps; steps [lo, hi] of each tile (hi < lo: no rows)
    int lo[kTiles], hi[kTiles], page0 = 0, steps = 0;
#pragma unroll
    for (int t = 0; t < kTiles; t++) {
        const unsigned b = m0 + t * kTileRows, e = min(packed, b + kTileRows);
        lo[t] = 0, hi[t] = -1;
        if (n > 0 && ok_seq && b < e) {
            const int from = start + (int)(b / (unsigned)group), to = start + (int)((e - 1) / (unsigned)group);
            const int first = a.window ? max(0, from - a.window + 1) / kPagePositions : 0;
            if (t == 0) page0 = first;
            lo[t] = (first - page0) / kPages;
            hi[t] = (to / kPagePositions - page0) / kPages;
            steps = max(steps, hi[t] + 1);
        }
    }
    // a warp's tile, and the steps it takes
    const auto pick = [&](const int(&x)[kTiles], int t) { return t == 0 ? x[0] : t == 1 ? x[1] : x[kTiles - 1]; };
    const int last_pos = start + (int)((max(1u, min(packed, m0 + kCtaRows)) - 1) / (unsigned)group);  // the CTA's last query

    if (warp < St::kConvertWarp) {
        // ------------------------------------------------------- softmax --
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(St::kSoftmaxRegs));
        const int t = warp >> 2, row = threadIdx.x & (kTileRows - 1);
        const int lo_t = pick(lo, t), hi_t = pick(hi, t);
        const unsigned m = m0 + t * kTileRows + row;
        const bool valid = m < packed;  // (no work: packed is 0)
        const int query = valid ? (int)(m / (unsigned)group) : 0;
        const int head = kv_head * group + (valid ? (int)(m - (unsigned)query * group) : 0);
        const size_t at = (size_t)(first_row + query);
        const int pos = start + query;
        float scale_q = 1.0f;
        if (hi_t >= lo_t) {
            // the query row: normalised to fp16 (in two parts), dims in the order the key tiles have them, into the
            // swizzled A tile.  A warp's rows come in whole sectors, through the tile's own place (thread = row would
            // take a line a lane and access; there and for the results that was 4 us of a CTA's 20).
            const uint64_t src = valid ? (uint64_t)(static_cast<const T *>(a.q) + at * a.q_stride + (size_t)head * kHeadDim) : 0;
#pragma unroll
            for (int i = 0; i < St::kRowChunks; i++) {
                const uint64_t from = __shfl_sync(0xffffffffu, src, St::chunk_row(i, lane));
                async_chunk(row_chunk(s, t, (warp & 3) * 32 + St::chunk_row(i, lane), lane % St::kRowChunks),
                            from ? reinterpret_cast<const uint8_t *>(from) + lane % St::kRowChunks * 16 : a.q, from != 0);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            float x[kHeadDim], peak = 0.0f;
#pragma unroll
            for (int j = 0; j < St::kRowChunks; j++) {
                constexpr int kPer = 16 / (int)sizeof(T);
                const uint4 w = *reinterpret_cast<const uint4 *>(row_chunk(s, t, row, j));
#pragma unroll
                for (int e = 0; e < kPer; e++) {
                    const float f = to_float(reinterpret_cast<const T *>(&w)[e]);
                    x[j * kPer + e] = f, peak = fmaxf(peak, fabsf(f));
                }
            }
            float up;
            query_norm(peak, up, scale_q);
#pragma unroll
            for (int j = 0; j < 8; j++) {  // 16-byte chunk j: dims d..d+3 and d+16..d+19
                const int d = (j >> 2) * 32 + (j & 3) * 4;
                const float f[8] = {x[d] * up,      x[d + 1] * up,  x[d + 2] * up,  x[d + 3] * up,
                                    x[d + 16] * up, x[d + 17] * up, x[d + 18] * up, x[d + 19] * up};
                uint4 h = make_uint4(half_pair(f[0], f[1]), half_pair(f[2], f[3]), half_pair(f[4], f[5]),
                                     half_pair(f[6], f[7]));
                const int byte = row * 128 + ((j ^ (row & 7)) << 4);
                *reinterpret_cast<uint4 *>(&s.q[t][0][byte]) = h;
                if constexpr (kSplit)
                    *reinterpret_cast<uint4 *>(&s.q[t][kSplit ? 1 : 0][byte]) =
                        make_uint4(half_rest(f[0], f[1], h.x), half_rest(f[2], f[3], h.y), half_rest(f[4], f[5], h.z),
                                   half_rest(f[6], f[7], h.w));
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.q_full);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + St::kS + t * kCols, to = tmem + lanes + St::kO + t * kHeadDim;
        const uint32_t tp = tmem + lanes + St::kP + t * St::kPCols;
        [[maybe_unused]] const uint32_t sum_at = tmem + lanes + St::kSum + t * kHeadDim;
        float top = -INFINITY, total = 0.0f;
        [[maybe_unused]] float owed = 1.0f;  // what O was scaled by since the last time it went over to the sum
        int exponent = kMinExponent;
        bool ok = true;
        for (int i = lo_t; ok && i <= hi_t; i++) {
            const int it = i - lo_t, st = i % kStages;
            // positions [from, upto] of the step are this row's
            const int upto = max(pos - (page0 + i * kPages) * kPagePositions, -1);
            const int from = a.window ? upto - a.window + 1 : 0;
            const bool whole = __all_sync(0xffffffffu, upto >= kCols - 1 && from <= 0);
            ok = warp_wait(&s.s_full[t], it & 1, &s.abort);
            if (!ok) break;
            tc_fence_after();
            uint32_t r[kCols];
#pragma unroll
            for (int c = 0; c < kCols; c += 32) tmem_ld32(ts + c, reinterpret_cast<uint32_t(&)[32]>(r[c]));
            const int ke = s.exponent[st];
            const float f = fminf(fmaxf(scale_q * s.key_factor[st], FLT_MIN), FLT_MAX);  // it multiplies infinities
            tmem_ld_wait(r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.s_free[t]);
            // has the previous product read P and finished O?  (asked ahead: the answer takes some 70 clocks)
            const bool pv_ready = it == 0 || mbar_test_wait(&s.pv_done[t], (it - 1) & 1);
            if constexpr (!St::kFold) {  // the key scales
                const ulonglong2 *ks = reinterpret_cast<const ulonglong2 *>(s.ks[st]);
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                    const ulonglong2 k2 = ks[j / 4];
                    float x[4];
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), k2.x), x[0], x[1]);
                    f2_unpack(f2_mul(f2_pack(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), k2.y), x[2], x[3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) r[j + e] = __float_as_uint(x[e]);
                }
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < kCols; j++)
                    if (j > upto || j < from) r[j] = __float_as_uint(-INFINITY);
            }
            float peaks[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < kCols; j += 2)
                peaks[(j >> 1) & 3] = fmaxf(peaks[(j >> 1) & 3], fmaxf(__uint_as_float(r[j]), __uint_as_float(r[j + 1])));
            const float peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3])) * f;
            float keep = 1.0f;
            if (peak - top > kLazy || (top == -INFINITY && peak > -INFINITY)) {
                keep = top == -INFINITY ? 0.0f : exp2_approx(top - peak);
                total *= keep;
                top = peak;
            }
            if (ke > exponent) keep *= exp2_approx((float)(exponent - ke));
            exponent = ke;
            // folded value scales leave P room up to 2^15
            const float base = (top == -INFINITY ? 0.0f : top) - (St::kFold ? 8.0f : 0.0f);
            [[maybe_unused]] const ulonglong2 *vs = reinterpret_cast<const ulonglong2 *>(s.vs[st]);
            const uint64_t f2 = f2_pack(f, f), base2 = f2_pack(-base, -base);
            uint64_t sums[2] = {0, 0};
            uint32_t hp[kCols / 2];
            [[maybe_unused]] uint32_t lp[kSplit ? kCols / 2 : 1];
#pragma unroll
            for (int j = 0; j < kCols; j += 4) {
                [[maybe_unused]] ulonglong2 v2;
                if constexpr (!St::kFold) v2 = vs[j / 4];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int k = j + 2 * u;
                    float e0, e1;
                    f2_unpack(f2_fma(f2_pack(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), f2, base2), e0, e1);
                    e0 = exp2_approx(e0), e1 = exp2_approx(e1);
                    const uint64_t e = f2_pack(e0, e1);
                    sums[u] = f2_add(sums[u], e);
                    if constexpr (!St::kFold) f2_unpack(f2_mul(e, u ? v2.y : v2.x), e0, e1);
                    hp[k / 2] = half_pair(e0, e1);
                    if constexpr (kSplit) lp[kSplit ? k / 2 : 0] = half_rest(e0, e1, hp[k / 2]);
                }
            }
            float sum0, sum1;
            f2_unpack(f2_add(sums[0], sums[1]), sum0, sum1);
            total += sum0 + sum1;
            if (!__all_sync(0xffffffffu, pv_ready)) {
                ok = warp_wait(&s.pv_done[t], (it - 1) & 1, &s.abort);
                if (!ok) break;
            }
            tc_fence_after();
            if (it > 0 && __any_sync(0xffffffffu, keep != 1.0f)) {
#pragma unroll
                for (int c = 0; c < kHeadDim; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(to + c, o);
                    tmem_ld_wait(o);
#pragma unroll
                    for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                    tmem_st16(to + c, o);
                }
                if constexpr (kSplit) owed *= keep;
            }
#pragma unroll
            for (int c = 0; c < kCols / 2; c += 16) {
                tmem_st16(tp + c, reinterpret_cast<const uint32_t(&)[16]>(hp[c]));
                if constexpr (kSplit) tmem_st16(tp + St::kLo + c, reinterpret_cast<const uint32_t(&)[16]>(lp[kSplit ? c : 0]));
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[t]);
            if constexpr (kSplit) {
                if ((it + 1) % St::kFlush == 0 && i < hi_t) {  // O goes over to the sum
                    ok = warp_wait(&s.pv_done[t], it & 1, &s.abort);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < kHeadDim; c += 16) {
                        uint32_t o[16], u[16];
                        tmem_ld16(to + c, o);
                        tmem_ld16(sum_at + c, u);  // (nothing yet at the first)
                        tmem_ld_wait(o);
                        tmem_ld_wait(u);
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            o[j] = __float_as_uint(__uint_as_float(o[j]) + (it >= St::kFlush ? __uint_as_float(u[j]) * owed : 0.0f));
                        tmem_st16(sum_at + c, o);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    owed = 1.0f;
                }
            }
        }
        // the rows' results
        if (hi_t >= lo_t) {
            ok = ok && warp_wait(&s.pv_done[t], (hi_t - lo_t) & 1, &s.abort);
            if (!ok) {
                s.abort = 1;
                if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusTimeout);
            }
            tc_fence_after();
            uint32_t r0[32], r1[32];
            tmem_ld32(to, r0);
            tmem_ld32(to + 32, r1);
            tmem_ld_wait(r0);
            tmem_ld_wait(r1);
            if (kSplit && hi_t - lo_t >= St::kFlush) {
#pragma unroll
                for (int c = 0; c < kHeadDim; c += 16) {
                    uint32_t u[16];
                    tmem_ld16(sum_at + c, u);
                    tmem_ld_wait(u);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        uint32_t &o = c < 32 ? r0[c + j] : r1[(c + j) & 31];
                        o = __float_as_uint(__uint_as_float(o) + __uint_as_float(u[j]) * owed);
                    }
                }
            }
            const float inverse = ok ? 1.0f / total : __int_as_float(0x7fc00000), back = pow2(exponent - 8);
            float x[64];
#pragma unroll
            for (int j = 0; j < 32; j++) {
                x[j] = __uint_as_float(r0[j]) * inverse * back;
                x[j + 32] = __uint_as_float(r1[j]) * inverse * back;
            }
            // through the queries' place, whose products have ended, to whole sectors again
#pragma unroll
            for (int j = 0; j < St::kRowChunks; j++)
                store16(reinterpret_cast<T *>(row_chunk(s, t, row, j)), x + j * (16 / (int)sizeof(T)));
            __syncwarp();
            const uint64_t dst = valid ? (uint64_t)(static_cast<T *>(a.out) + at * a.out_stride + (size_t)head * kHeadDim) : 0;
#pragma unroll
            for (int i = 0; i < St::kRowChunks; i++) {
                const uint64_t to = __shfl_sync(0xffffffffu, dst, St::chunk_row(i, lane));
                const uint4 w = *reinterpret_cast<const uint4 *>(
                    row_chunk(s, t, (warp & 3) * 32 + St::chunk_row(i, lane), lane % St::kRowChunks));
                if (to) reinterpret_cast<uint4 *>(to)[lane % St::kRowChunks] = w;
            }
        } else if (valid) {  // a bad sequence
            if (a.c.status) atomicOr(a.c.status, kStatusBadPage);
            float x[64];
#pragma unroll
            for (int j = 0; j < 64; j++) x[j] = __int_as_float(0x7fc00000);
            T *dst = static_cast<T *>(a.out) + at * a.out_stride + (size_t)head * kHeadDim;
#pragma unroll
            for (int j = 0; j < 64; j += 16 / (int)sizeof(T)) store16(dst + j, x + j);
        }
    } else if (warp < kMmaWarp) {
        // -------------------------------------------------- page converter --
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(St::kConvertRegs));
        const int c = warp - St::kConvertWarp;
        int exponent = kMinExponent;
        const float fold = a.scale * kLog2E;
        for (int i = 0; i < steps; i++) {
            const int st = i % kStages, rs = i % St::kRaw;
            if (!warp_wait(&s.raw_full[rs], (i / St::kRaw) & 1, &s.abort) ||
                (i >= kStages && !warp_wait(&s.kv_empty[st], ((i / kStages) - 1) & 1, &s.abort))) {
                if (lane == 0 && !s.abort && a.c.status) atomicOr(a.c.status, kStatusTimeout);
                s.abort = 1;
                break;
            }
            // The scales, lane -> positions lane and lane + 32: those behind the CTA's last query belong to no one, the
            // keys' of a missing page are NaN, and those of a position whose value scale is no number.
            const int missing = s.missing[rs];
            float ks[kPages][2], vs[kPages][2];
            int key_top = 0, value_top = 0;
#pragma unroll
            for (int g = 0; g < kPages; g++) {
                const int seen = last_pos - (page0 + i * kPages + g) * kPagePositions;
                const uint8_t *rec = s.raw[rs][g];
                if ((missing >> g & 1) && c == 0 && lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int p = lane + 32 * h;
                    float k = reinterpret_cast<const float *>(rec + kKScaleOffset)[k_scale_index(p)] * fold;
                    float v = reinterpret_cast<const float *>(rec + kVScaleOffset)[v_scale_index(p)];
                    if ((missing >> g & 1) || !(fabsf(v) <= FLT_MAX)) k = __int_as_float(0x7fc00000), v = 0.0f;
                    if (p > seen) k = 0.0f, v = 0.0f;
                    ks[g][h] = k, vs[g][h] = v;
                    key_top = max(key_top, scale_exponent(k)), value_top = max(value_top, scale_exponent(v));
                }
            }
            const int key_exponent = max(kMinExponent, __reduce_max_sync(0xffffffffu, key_top) - 126);
            exponent = max(exponent, __reduce_max_sync(0xffffffffu, value_top) - 126);
            const float key_norm = pow2(8 - key_exponent), value_norm = pow2(8 - exponent);  // exponents in [-110, 128]
            if (c == 0 && lane == 0) s.key_factor[st] = pow2(key_exponent - 8), s.exponent[st] = exponent;
#pragma unroll
            for (int g = 0; g < kPages; g++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int p = lane + 32 * h;
                    const float k = ks[g][h] * key_norm, v = vs[g][h] * value_norm;
                    if constexpr (St::kFold) {  // the key scale as two fp16, the value scale as one
                        const uint32_t kh = half_pair(k, 0.0f);
                        reinterpret_cast<uint32_t *>(s.scales[c][0][g])[p] = half_pair(k, k - __low2float(as_half2(kh)));
                        reinterpret_cast<__half *>(s.scales[c][1][g])[p] = __float2half_rn(v);
                    } else {
                        if (c == 0) s.ks[st][g * kPagePositions + p] = k, s.vs[st][g * kPagePositions + p] = v;
                    }
                }
            __syncwarp();
            // A warp takes 16 positions of a page's keys and 16 dims of its values: two 512-byte blocks of each.
            uint4 kw[kPages][2], vw[kPages][2];
#pragma unroll
            for (int g = 0; g < kPages; g++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    // keys: lane -> row lane & 7 (and + 8), 4-dim column lane >> 3 of dims 32 u ..; values: lane -> dim
                    // lane & 7, positions 16 (lane >> 3) ..
                    const uint8_t *rec = s.raw[rs][g];
                    kw[g][u] = *reinterpret_cast<const uint4 *>(rec + (2 * c + u) * 512 + ((lane & 7) * 4 + (lane >> 3)) * 16);
                    const int d = (2 * c + u) * 8 + (lane & 7);
                    vw[g][u] = *reinterpret_cast<const uint4 *>(rec + kVOffset + d * 64 + (((lane >> 3) ^ ((d >> 1) & 3)) << 4));
                }
#pragma unroll
            for (int g = 0; g < kPages; g++) {
                const int row = c * 16 + (lane & 7);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t sh = 0, sl = 0;
                    if constexpr (St::kFold) {
                        const uint32_t sc = reinterpret_cast<const uint32_t *>(s.scales[c][0][g])[row + 8 * h];
                        sh = __byte_perm(sc, 0, 0x1010), sl = __byte_perm(sc, 0, 0x3232);
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        // words: (row, dims), (row + 8, dims), then dims + 16
                        const uint32_t w0 = h ? kw[g][u].y : kw[g][u].x, w1 = h ? kw[g][u].w : kw[g][u].z;
                        const int at = (row + 8 * h) * 128 + (((u * 4 + (lane >> 3)) ^ (row & 7)) << 4);
                        uint32_t x[4];
                        if constexpr (St::kFold) {
                            folded_codes(w0, sh, sl, x[0], x[1]);
                            folded_codes(w1, sh, sl, x[2], x[3]);
                        } else {
                            codes_to_half(w0, x[0], x[1]);
                            codes_to_half(w1, x[2], x[3]);
                        }
                        *reinterpret_cast<uint4 *>(&s.k[st][g][at]) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                uint32_t f[8];
                if constexpr (St::kFold) {
                    const uint4 *sc = reinterpret_cast<const uint4 *>(s.scales[c][1][g]) + (lane >> 3) * 2;
                    const uint4 s0 = sc[0], s1 = sc[1];
                    f[0] = s0.x, f[1] = s0.y, f[2] = s0.z, f[3] = s0.w, f[4] = s1.x, f[5] = s1.y, f[6] = s1.z, f[7] = s1.w;
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t words[4] = {vw[g][u].x, vw[g][u].y, vw[g][u].z, vw[g][u].w};
                    uint32_t h[8];
#pragma unroll
                    for (int j = 0; j < 4; j++) codes_to_half(words[j], h[2 * j], h[2 * j + 1]);
                    if constexpr (St::kFold) {
#pragma unroll
                        for (int j = 0; j < 8; j++) h[j] = half2_bits(__hmul2(as_half2(h[j]), as_half2(f[j])));
                    }
                    const int d = (2 * c + u) * 8 + (lane & 7), j = (lane >> 3) * 2;
                    *reinterpret_cast<uint4 *>(&s.v[st][g][d * 128 + ((j ^ (d & 7)) << 4)]) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(&s.v[st][g][d * 128 + (((j + 1) ^ (d & 7)) << 4)]) =
                        make_uint4(h[4], h[5], h[6], h[7]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.kv_full[st]);
        }
    } else {
        // ------------------------------------------------------ MMA issuer --
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(St::kMmaRegs));
        bool ok = true;
        if (warp == St::kCopyWarp) {
            // the records of each step into their ring, once the converters have read the step kRaw before
            const int page_end = last_pos / kPagePositions + 1;
            int ids = -1, i = 0;
            for (; i < steps; i++) {
                const int rs = i % St::kRaw;
                int absent = 0, found = 0, id[kPages];
#pragma unroll
                for (int g = 0; g < kPages; g++) {
                    const int rel = i * kPages + g, page = page0 + rel;
                    if ((rel & 31) == 0) ids = page + lane < page_end ? cache_page(a.c, slot, page + lane) : -1;
                    id[g] = __shfl_sync(0xffffffffu, ids, rel & 31);
                    if (id[g] >= 0) found++;
                    else if (page < page_end) absent |= 1 << g;  // behind the last page there is nothing to miss
                }
                if (i >= St::kRaw) {
                    const int j = i - St::kRaw;
                    ok = warp_wait(&s.kv_full[j % kStages], (j / kStages) & 1, &s.abort);
                    if (!ok) break;
                }
                if (lane == 0) {
                    s.missing[rs] = absent;
                    if (found) mbar_arrive_expect_tx(&s.raw_full[rs], found * kKvBlockBytes);
                    else mbar_arrive(&s.raw_full[rs]);
#pragma unroll
                    for (int g = 0; g < kPages; g++)
                        if (id[g] >= 0)
                            bulk_g2s(s.raw[rs][g], cache_record(a.c, id[g], kv_head), kKvBlockBytes, &s.raw_full[rs]);
                }
                __syncwarp();
            }
            // every copy in flight lands before the CTA exits (bounded)
            if (!ok)
                for (int j = max(0, i - St::kRaw); j < i; j++)
                    mbar_wait_bounded(&s.raw_full[j % St::kRaw], (j / St::kRaw) & 1, kPromptWait);
        } else if (warp < kMmaWarp + kTiles) {
            // A warp issues the products of one tile.
            constexpr uint32_t idesc_s = idesc_f16(kTileRows, kCols), idesc_o = idesc_f16(kTileRows, kHeadDim);
            const int t = warp - kMmaWarp, lo_t = pick(lo, t), hi_t = pick(hi, t);
            const uint32_t ts = tmem + St::kS + t * kCols, to = tmem + St::kO + t * kHeadDim, tp = tmem + St::kP + t * St::kPCols;
            auto scores = [&](int i) {
                if (!ok || i < lo_t || i > hi_t) return;
                const int it = i - lo_t, st = i % kStages;
                ok = warp_wait(&s.kv_full[st], (i / kStages) & 1, &s.abort) &&
                     (it == 0 || warp_wait(&s.s_free[t], (it - 1) & 1, &s.abort));
                if (!ok) return;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < St::kQParts; i++) {  // the small part first: the accumulator truncates what is added
                    const uint64_t q = sw128_kmajor_desc(s.q[t][St::kQParts - 1 - i]), b = sw128_kmajor_desc(s.k[st]);
#pragma unroll
                    for (int k = 0; k < 4; k++) mma_f16_ss(ts, q + 2 * k, b + 2 * k, idesc_s, i + k > 0);
                }
                // the products' end, and (by a plain arrive) the converters' scales of the step, which this warp has seen
                mma_commit_elect(&s.s_full[t]);
                if (lane == 0) mbar_arrive(&s.s_full[t]);
            };
            if (steps > 0) ok = warp_wait(&s.q_full, 0, &s.abort);
            scores(0);
            for (int i = 0; i < steps && ok; i++) {
                scores(i + 1);
                const int it = i - lo_t, st = i % kStages;
                if (i >= lo_t && i <= hi_t) {
                    ok = ok && warp_wait(&s.p_full[t], it & 1, &s.abort);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int i = 0; i < (kSplit ? 2 : 1); i++)  // the small part first
#pragma unroll
                        for (int k = 0; k < 4 * kPages; k++)
                            mma_f16_ts(to, tp + (kSplit && i == 0 ? St::kLo : 0) + k * 8,
                                       sw128_kmajor_desc(s.v[st][k >> 2]) + 2 * (k & 3), idesc_o,
                                       (kSplit ? it % St::kFlush : it) + i + k > 0);
                    mma_commit_elect(&s.pv_done[t]);
                } else {  // the step is other tiles' alone
                    ok = warp_wait(&s.kv_full[st], (i / kStages) & 1, &s.abort);
                    if (!ok) break;
                }
                if (i + kStages < steps) mma_commit_elect(&s.kv_empty[st]);  // (no arrival that nobody waits for)
            }
            if (!ok) {  // every product in flight ends before the CTA's TMEM is freed (bounded)
                mma_commit_elect(&s.drained[t]);
                mbar_wait_bounded(&s.drained[t], 0, kPromptWait);
            }
        }
        if (!ok) {
            s.abort = 1;
            if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusTimeout);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

}  // namespace

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
        using T = decltype(t);
        const auto kernel = attention_prompt_kernel<T>;
        // each sequence ends one tile early at most: no more tiles than these, whatever the lengths are
        const long long tiles = (long long)rows * (heads / kv_heads) / Step<T>::kRows + sequences;
        NDL_REQUIRE(tiles * kv_heads <= 0x7FFFFFFFLL, "%d rows of %d heads in %d sequences: too many", rows, heads,
                    sequences);
        constexpr size_t smem = sizeof(PromptSmem<T>) + 1024;
        static DeviceOnce attribute;  // the attribute belongs to the kernel on one device
        const int st = attribute.run([&] {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            return e == cudaSuccess ? (int)NDL_OK
                                    : set_error(NDL_ERR_CUDA, "prompt attention smem: %s", cudaGetErrorString(e));
        });
        if (st != NDL_OK) return st;
        kernel<<<(unsigned)(tiles * kv_heads), Step<T>::kThreads, smem, (cudaStream_t)stream>>>(a);
        return check_launch("attention_prompt");
    });
}
