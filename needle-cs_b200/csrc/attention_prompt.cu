// Whole-prompt attention over the paged int8 cache, on the fifth-generation
// tensor cores.
//
// A CTA takes 256 packed rows (two tiles of 128) of one sequence and kv head;
// packed row m is query m / group of the sequence and query head m % group of
// the kv head's group, so a page of keys and values serves every query head
// that shares it.  It walks the pages its rows see, one page of 64 positions
// a step, with the softmax's running maximum and sum:
//   S = Q K^T       tcgen05.mma, fp16 operands, fp32 accumulator in TMEM
//   t = S ks_j      (ks: the key scales, with scale * log2 e folded in)
//   e = 2^(q (t - m)),  l += e,  P = e vs_j,  O += P V
// q, a power of two per row, brings the row's largest query to [2^10, 2^11),
// so 16-bit queries are exact in fp16; key and value codes are small integers,
// exact too.  P rounds to fp16 (half a step, 2^-11, as an fp16 result does);
// fp32 callers get queries and P as two fp16 parts each (22 bits) and twice
// the products.  So that P fits fp16 whatever the value scales are, they are
// divided by 2^k, k the exponent of the largest seen so far (O is rescaled
// where it grows), and m follows the true maximum only where that is 7 binary
// orders above it: P <= 2^7 2^8, and O is rescaled on few pages.
//
// Warps: 4 softmax warps a tile (thread = row, so maximum and sum need no
// exchange), 4 that convert pages (int8 in global memory -> fp16 tiles in
// shared memory, 128-byte swizzled rows), 1 that issues every MMA.  P goes
// back to TMEM, from where the second product takes it as its A operand.
#include "attention_math.cuh"
#include "tc.cuh"

namespace ndl {

namespace {

constexpr int kTileRows = 128;                 // MMA rows: TMEM lanes
constexpr int kCtaRows = 2 * kTileRows;
constexpr int kStages = 4;                     // converted pages in flight
constexpr int kPromptThreads = 13 * 32;
constexpr int kConvertWarp = 8, kMmaWarp = 12;
constexpr int kTileBytes = kTileRows * kHeadDim * 2;   // 16 KB of queries
constexpr int kPageTile = kPagePositions * kHeadDim * 2;  // 8 KB of keys or values
constexpr uint32_t kPromptWait = 1u << 22;     // waits of about a microsecond: a few seconds
// TMEM columns: scores, outputs, probabilities (two fp16 a column) of both tiles
constexpr int kColS = 0, kColO = 128, kColP = 256, kColLo = 64;
constexpr int kTmemCols = 512;

struct PromptArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int32_t *seq_rows, *seq_slot, *seq_pos;
    int rows, sequences, heads, window;
    float scale;
    PagedCache c;
};

template <bool kSplit>
struct PromptSmem {
    uint8_t q[2][kSplit ? 2 : 1][kTileBytes];  // 1024-byte aligned
    uint8_t k[kStages][kPageTile], v[kStages][kPageTile];
    float ks[kStages][kPagePositions], vs[kStages][kPagePositions];
    int exponent[kStages];
    uint64_t kv_full[kStages], kv_empty[kStages];
    uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
    uint32_t tmem;
    int seq, tile;  // this CTA's work: sequence (-1: none) and 256-row tile of it
    volatile int abort;
};

// kind::f16, fp32 accumulator, A and B fp16, both K-major.
constexpr uint32_t idesc_f16(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
        "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <class T, bool kSplit>
__global__ void __launch_bounds__(kPromptThreads, 1) attention_prompt_kernel(PromptArgs a) {
    extern __shared__ uint8_t smem_raw[];
    PromptSmem<kSplit> &s = *reinterpret_cast<PromptSmem<kSplit> *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                                     ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv_head = blockIdx.x % a.c.heads, work = blockIdx.x / a.c.heads;
    const int group = a.heads / a.c.heads;

    // This CTA's tile: sequences hold ceil(rows * group / 256) tiles each.
    if (warp == 0) {
        int seq = -1, tile = 0, before = 0;
        for (int base = 0; base < a.sequences && seq < 0; base += 32) {
            const int i = base + lane;
            int tiles = 0;
            if (i < a.sequences) {
                const int b = a.seq_rows[i], e = a.seq_rows[i + 1];
                if (b >= 0 && e >= b && e <= a.rows) tiles = (int)(((long long)(e - b) * group + kCtaRows - 1) / kCtaRows);
            }
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const bool mine = work >= before + sum - tiles && work < before + sum;
            const unsigned who = __ballot_sync(0xffffffffu, mine);
            if (who) {
                const int l = __ffs(who) - 1;
                seq = base + l;
                // the last tile, which sees the most pages, first
                tile = __shfl_sync(0xffffffffu, tiles - 1 - (work - (before + sum - tiles)), l);
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) s.seq = seq, s.tile = tile, s.abort = 0;
        if (blockIdx.x == 0)
            for (int i = lane; i < a.sequences; i += 32) {
                const int b = a.seq_rows[i], e = a.seq_rows[i + 1];
                if ((b < 0 || e < b || e > a.rows) && a.c.status) atomicOr(a.c.status, kStatusBadPage);
            }
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            for (int i = 0; i < kStages; i++) mbar_init(&s.kv_full[i], 4), mbar_init(&s.kv_empty[i], 1);
            for (int t = 0; t < 2; t++)
                mbar_init(&s.s_full[t], 1), mbar_init(&s.s_free[t], 4), mbar_init(&s.p_full[t], 4),
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
    const int seq = s.seq;
    const int first_row = seq >= 0 ? a.seq_rows[seq] : 0;
    const int n = seq >= 0 ? a.seq_rows[seq + 1] - first_row : 0;
    const int slot = seq >= 0 ? a.seq_slot[seq] : 0, start = seq >= 0 ? a.seq_pos[seq] : 0;
    const bool ok_seq = slot >= 0 && slot < a.c.slots && start >= 0 &&
                        (long long)start + n <= (long long)a.c.max_pages * kPagePositions;
    const long long packed = (long long)n * group, m0 = (long long)s.tile * kCtaRows;
    // pages [lo, hi] of each tile (hi < lo: no rows)
    int lo[2], hi[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const long long b = m0 + t * kTileRows, e = min(packed, b + kTileRows);
        lo[t] = 0, hi[t] = -1;
        if (seq >= 0 && ok_seq && b < e) {
            const int from = start + (int)(b / group), to = start + (int)((e - 1) / group);
            lo[t] = a.window ? max(0, from - a.window + 1) / kPagePositions : 0;
            hi[t] = to / kPagePositions;
        }
    }
    const int page0 = lo[0], page1 = max(hi[0], hi[1]);
    const int last_pos = start + (int)((min(packed, m0 + kCtaRows) - 1) / group);  // the CTA's last query

    if (warp < kConvertWarp) {
        // ------------------------------------------------------- softmax --
        const int t = warp >> 2, row = threadIdx.x & (kTileRows - 1);
        const long long m = m0 + t * kTileRows + row;
        const bool valid = seq >= 0 && m < packed;
        const int query = valid ? (int)(m / group) : 0, head = kv_head * group + (valid ? (int)(m % group) : 0);
        const size_t at = (size_t)(first_row + query);
        const int pos = start + query;
        float scale_q = 1.0f;
        if (hi[t] >= lo[t]) {
            // the query row: normalised to fp16 (in two parts), dims in the
            // order the key tiles have them, into the swizzled A tile
            const T *src = static_cast<const T *>(a.q) + at * a.q_stride + (size_t)head * kHeadDim;
            float x[kHeadDim], peak = 0.0f;
#pragma unroll
            for (int i = 0; i < kHeadDim; i += 4) {
                float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (valid) load4(src + i, f);
#pragma unroll
                for (int j = 0; j < 4; j++) x[i + j] = f[j], peak = fmaxf(peak, fabsf(f[j]));
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
        __syncthreads();
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + kColS + t * 64, to = tmem + lanes + kColO + t * 64;
        const uint32_t tp = tmem + lanes + kColP + t * 32;
        float top = -INFINITY, total = 0.0f;
        int exponent = kMinExponent;
        bool ok = true;
        for (int i = lo[t]; i <= hi[t]; i++) {
            const int it = i - lo[t], st = (i - page0) % kStages;
            ok = mbar_wait_bounded(&s.s_full[t], it & 1, kPromptWait) &&
                 mbar_wait_bounded(&s.kv_full[st], ((i - page0) / kStages) & 1, kPromptWait);
            if (!__all_sync(0xffffffffu, ok) || s.abort) break;
            tc_fence_after();
            uint32_t r0[32], r1[32];
            tmem_ld32(ts, r0);
            tmem_ld32(ts + 32, r1);
            tmem_ld_wait(r0);
            tmem_ld_wait(r1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.s_free[t]);
            float x[64];
            const float4 *ks = reinterpret_cast<const float4 *>(s.ks[st]);
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                const float4 c = ks[j >> 2];
                const uint32_t *r = j < 32 ? r0 + j : r1 + (j - 32);
                x[j] = __uint_as_float(r[0]) * c.x, x[j + 1] = __uint_as_float(r[1]) * c.y;
                x[j + 2] = __uint_as_float(r[2]) * c.z, x[j + 3] = __uint_as_float(r[3]) * c.w;
            }
            // positions this row does not see
            const int upto = pos - i * kPagePositions;
            const int from = a.window ? upto - a.window + 1 : 0;
            const bool whole = __all_sync(0xffffffffu, upto >= kPagePositions - 1 && from <= 0);
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 64; j++)
                    if (j > upto || j < from) x[j] = -INFINITY;
            }
            float peak = x[0];
#pragma unroll
            for (int j = 1; j < 64; j++) peak = fmaxf(peak, x[j]);
            const int ke = s.exponent[st];
            float keep = 1.0f;
            const bool grew = (peak - top) * scale_q > kLazy || (top == -INFINITY && peak > -INFINITY);
            if (grew) {
                keep = exp2_approx((top - peak) * scale_q);
                if (top == -INFINITY) keep = 0.0f;
                total *= keep;
                top = peak;
            }
            if (ke > exponent) keep *= exp2_approx((float)(exponent - ke));
            exponent = ke;
            const float base = top == -INFINITY ? 0.0f : top * scale_q;
            uint32_t hp[32], lp[kSplit ? 32 : 1];
            const float4 *vs = reinterpret_cast<const float4 *>(s.vs[st]);
            float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                const float4 c = vs[j >> 2];
                float e[4], p[4];
#pragma unroll
                for (int u = 0; u < 4; u++) e[u] = exp2_approx(fmaf(x[j + u], scale_q, -base));
                sum0 += e[0] + e[2], sum1 += e[1] + e[3];
                p[0] = e[0] * c.x, p[1] = e[1] * c.y, p[2] = e[2] * c.z, p[3] = e[3] * c.w;
                if (!whole) {
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        if (j + u > upto || j + u < from) p[u] = 0.0f;
                }
                hp[j >> 1] = half_pair(p[0], p[1]), hp[(j >> 1) + 1] = half_pair(p[2], p[3]);
                if constexpr (kSplit)
                    lp[kSplit ? j >> 1 : 0] = half_rest(p[0], p[1], hp[j >> 1]),
                    lp[kSplit ? (j >> 1) + 1 : 0] = half_rest(p[2], p[3], hp[(j >> 1) + 1]);
            }
            total += sum0 + sum1;
            // the previous product has read P and finished O
            if (it > 0) {
                ok = mbar_wait_bounded(&s.pv_done[t], (it - 1) & 1, kPromptWait);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc_fence_after();
                if (__any_sync(0xffffffffu, keep != 1.0f)) {
                    tmem_ld32(to, r0);
                    tmem_ld32(to + 32, r1);
                    tmem_ld_wait(r0);
                    tmem_ld_wait(r1);
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        r0[j] = __float_as_uint(__uint_as_float(r0[j]) * keep);
                        r1[j] = __float_as_uint(__uint_as_float(r1[j]) * keep);
                    }
                    tmem_st32(to, r0);
                    tmem_st32(to + 32, r1);
                }
            }
            tmem_st32(tp, hp);
            if constexpr (kSplit) tmem_st32(tp + kColLo, reinterpret_cast<const uint32_t(&)[32]>(lp));
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.p_full[t]);
        }
        // the rows' results
        if (hi[t] >= lo[t]) {
            ok = ok && !s.abort && mbar_wait_bounded(&s.pv_done[t], (hi[t] - lo[t]) & 1, kPromptWait);
            ok = __all_sync(0xffffffffu, ok);
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
            if (valid) {
                const float inverse = ok ? 1.0f / total : __int_as_float(0x7fc00000), back = pow2(exponent - 8);
                float x[64];
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    x[j] = __uint_as_float(r0[j]) * inverse * back;
                    x[j + 32] = __uint_as_float(r1[j]) * inverse * back;
                }
                T *dst = static_cast<T *>(a.out) + at * a.out_stride + (size_t)head * kHeadDim;
#pragma unroll
                for (int j = 0; j < 64; j += 16 / (int)sizeof(T)) store16(dst + j, x + j);
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
        const int c = warp - kConvertWarp;
        int exponent = kMinExponent;
        int ids = 0;
        struct Page {
            uint4 k[2], v[2];
            float2 scale;
            int id;
        } cur, nxt;
        const float fold = a.scale * kLog2E;
        auto fetch = [&](int i, Page &p) {
            const int rel = i - page0;
            if ((rel & 31) == 0) ids = i + lane <= page1 ? cache_page(a.c, slot, i + lane) : -1;
            p.id = __shfl_sync(0xffffffffu, ids, rel & 31);
            if (p.id < 0) return;
            const uint8_t *rec = cache_record(a.c, p.id, kv_head);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                // keys: lane -> (row & 7 = lane & 7, 4-dim column lane >> 3) of a 512-byte block; values: dim and 16
                // positions
                p.k[u] = __ldg(reinterpret_cast<const uint4 *>(rec + (c * 2 + u) * 512 + ((lane & 7) * 4 + (lane >> 3)) * 16));
                const int d = (c * 2 + u) * 8 + (lane & 7);
                p.v[u] = __ldg(reinterpret_cast<const uint4 *>(rec + kVOffset + d * 64 + (((lane >> 3) ^ ((d >> 1) & 3)) << 4)));
            }
            if (c == 0) {  // key scales of positions lane, lane + 32
                p.scale.x = __ldg(reinterpret_cast<const float *>(rec + kKScaleOffset) + k_scale_index(lane));
                p.scale.y = __ldg(reinterpret_cast<const float *>(rec + kKScaleOffset) + k_scale_index(lane + 32));
            } else if (c == 1) {
                p.scale.x = __ldg(reinterpret_cast<const float *>(rec + kVScaleOffset) + lane);
                p.scale.y = __ldg(reinterpret_cast<const float *>(rec + kVScaleOffset) + lane + 32);
            }
        };
        if (page0 <= page1) fetch(page0, cur);
        __syncthreads();
        for (int i = page0; i <= page1; i++) {
            if (i < page1) fetch(i + 1, nxt);
            const int rel = i - page0, st = rel % kStages;
            if (rel >= kStages) {
                const bool ok = mbar_wait_bounded(&s.kv_empty[st], ((rel / kStages) - 1) & 1, kPromptWait);
                if (!__all_sync(0xffffffffu, ok) || s.abort) {
                    s.abort = 1;
                    if (lane == 0 && !ok && a.c.status) atomicOr(a.c.status, kStatusTimeout);
                    break;
                }
            }
            const bool there = cur.id >= 0;
            if (!there) {
#pragma unroll
                for (int u = 0; u < 2; u++) cur.k[u] = cur.v[u] = make_uint4(0, 0, 0, 0);
                if (lane == 0 && c == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int block = c * 2 + u;  // (16-row tile, 32-dim step)
                const int row = (block >> 1) * 16 + (lane & 7), j = (block & 1) * 4 + (lane >> 3);
                uint4 a0, a1;
                codes_to_half(cur.k[u].x, a0.x, a0.y);
                codes_to_half(cur.k[u].z, a0.z, a0.w);
                codes_to_half(cur.k[u].y, a1.x, a1.y);
                codes_to_half(cur.k[u].w, a1.z, a1.w);
                const int byte = row * 128 + ((j ^ (row & 7)) << 4);
                *reinterpret_cast<uint4 *>(&s.k[st][byte]) = a0;
                *reinterpret_cast<uint4 *>(&s.k[st][byte + 8 * 128]) = a1;
                const int d = block * 8 + (lane & 7), jv = (lane >> 3) * 2;
                codes_to_half(cur.v[u].x, a0.x, a0.y);
                codes_to_half(cur.v[u].y, a0.z, a0.w);
                codes_to_half(cur.v[u].z, a1.x, a1.y);
                codes_to_half(cur.v[u].w, a1.z, a1.w);
                *reinterpret_cast<uint4 *>(&s.v[st][d * 128 + ((jv ^ (d & 7)) << 4)]) = a0;
                *reinterpret_cast<uint4 *>(&s.v[st][d * 128 + (((jv + 1) ^ (d & 7)) << 4)]) = a1;
            }
            // scales; those behind the CTA's last query belong to no one
            const int seen = last_pos - i * kPagePositions;
            float2 f = cur.scale;
            if (!there) f.x = f.y = __int_as_float(0x7fc00000);
            if (lane > seen) f.x = 0.0f;
            if (lane + 32 > seen) f.y = 0.0f;
            if (c == 0) {
                s.ks[st][lane] = f.x * fold;
                s.ks[st][lane + 32] = f.y * fold;
            } else if (c == 1) {
                if (!there) f.x = f.y = 0.0f;
                const int e = __reduce_max_sync(0xffffffffu, max(scale_exponent(f.x), scale_exponent(f.y)));
                exponent = max(exponent, e - 126);
                const float down = pow2(8 - exponent);  // -110 <= exponent <= 128
                s.vs[st][lane] = f.x * down;
                s.vs[st][lane + 32] = f.y * down;
                if (lane == 0) s.exponent[st] = exponent;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.kv_full[st]);
            cur = nxt;
        }
    } else {
        // ------------------------------------------------------ MMA issuer --
        __syncthreads();
        if (lane == 0 && page0 <= page1) {
            const uint32_t idesc = idesc_f16(kTileRows, kPagePositions);
            bool ok = true;
            auto scores = [&](int t, int i) {
                if (!ok || i < lo[t] || i > hi[t]) return;
                const int it = i - lo[t], rel = i - page0, st = rel % kStages;
                ok = mbar_wait_bounded(&s.kv_full[st], (rel / kStages) & 1, kPromptWait) &&
                     (it == 0 || mbar_wait_bounded(&s.s_free[t], (it - 1) & 1, kPromptWait));
                if (!ok) return;
                tc_fence_after();
                const uint64_t b = sw128_kmajor_desc(s.k[st]);
#pragma unroll
                for (int part = 0; part < (kSplit ? 2 : 1); part++) {
                    const uint64_t q = sw128_kmajor_desc(s.q[t][part]);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_f16_ss(tmem + kColS + t * 64, q + 2 * k, b + 2 * k, idesc, part + k > 0);
                }
                mma_commit(&s.s_full[t]);
            };
            auto values = [&](int t, int i) {
                if (!ok || i < lo[t] || i > hi[t]) return;
                const int it = i - lo[t], st = (i - page0) % kStages;
                ok = mbar_wait_bounded(&s.p_full[t], it & 1, kPromptWait);
                if (!ok) return;
                tc_fence_after();
                const uint64_t b = sw128_kmajor_desc(s.v[st]);
#pragma unroll
                for (int part = 0; part < (kSplit ? 2 : 1); part++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_f16_ts(tmem + kColO + t * 64, tmem + kColP + t * 32 + part * kColLo + k * 8, b + 2 * k,
                                   idesc, it + part + k > 0);
                mma_commit(&s.pv_done[t]);
            };
            scores(0, page0);
            scores(1, page0);
            for (int i = page0; i <= page1 && ok && !s.abort; i++) {
                scores(0, i + 1);
                scores(1, i + 1);
                values(0, i);
                values(1, i);
                if (ok) mma_commit(&s.kv_empty[(i - page0) % kStages]);
            }
            if (!ok) {
                s.abort = 1;
                if (a.c.status) atomicOr(a.c.status, kStatusTimeout);
            }
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
    // each sequence ends one tile early at most: no more tiles than these, whatever the lengths are
    const long long tiles = (long long)rows * (heads / kv_heads) / kCtaRows + sequences;
    NDL_REQUIRE(tiles * kv_heads <= 0x7FFFFFFFLL, "%d rows of %d heads in %d sequences: too many", rows, heads,
                sequences);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr bool kSplit = sizeof(T) == 4;
        const auto kernel = attention_prompt_kernel<T, kSplit>;
        constexpr size_t smem = sizeof(PromptSmem<kSplit>) + 1024;
        static DeviceOnce attribute;  // the attribute belongs to the kernel on one device
        const int st = attribute.run([&] {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            return e == cudaSuccess ? (int)NDL_OK
                                    : set_error(NDL_ERR_CUDA, "prompt attention smem: %s", cudaGetErrorString(e));
        });
        if (st != NDL_OK) return st;
        kernel<<<(unsigned)(tiles * kv_heads), kPromptThreads, smem, (cudaStream_t)stream>>>(a);
        return check_launch("attention_prompt");
    });
}
