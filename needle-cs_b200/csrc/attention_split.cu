// Attention of single tokens over the paged int8 cache, split over its length.
//
// A row's query heads that share a kv head (at most 16 at a time) attend
// together; such an item reads one 8704-byte record per page.  All records of
// a call, item after item, are dealt out evenly over one CTA an SM, and each
// CTA's over its warps, whatever the rows' lengths are: one long row fills the
// card as well as many ragged ones.  A warp streams its records through its
// own ring in shared memory (one bulk copy each, 11 warps x 2 records = 191 KB
// an SM; warps count, for the arithmetic, more than bytes in flight: when 8 warps
// x 3 records took 239 us, 12 x 2 took 215) and keeps a running maximum, sum and
// output per head:
//   S = Q K^T, O += (e vs) V   mma.sync m16n8k16, positions (then dims) as rows;
// the codes become fp16 exactly in registers, from the fragments the pages
// hold.  Tensor cores because a position costs 128 products a head and 128
// conversions, and a kv head's group shares the conversions; tcgen05 would
// need tiles of 128 rows, and there are at most 16.
// An item inside one warp is finished there.  Pieces of the others (O / l, m,
// l) meet in shared memory; those of items that reach over a CTA's records go
// to the workspace, and a second kernel, launched early, joins them.  Pieces
// are always taken in record order, so the result does not depend on timing.
// A few items (one an SM) of a few pages take a CTA each instead: no look at the
// other rows and no second kernel (8 kv heads, fp32, split and whole: 1 row of 4
// pages 10.6 and 6.8 us, of 16 11.1 and 11.2, of 24 11.2 and 13.4; 18 rows of up
// to 4 pages 11.2 and 7.2, 16 16.8 and 11.6, 24 17.0 and 14.2; bf16: of 16 pages
// 10.6 and 10.1, 12.9 and 10.4).
//
// Bound by memory where the cache is long: 256 rows of up to 8192 positions, 8
// kv heads, bf16: 194 us (5.6 TB/s, floor 167); heads as the products' columns, of
// which there are 8, cost half of what they cost as their 16 rows (217 us).  One
// row of 100003 positions: 34 us (floor 17), of which some 10 are the launch, the
// look at the rows and the join.  64 sessions, fp32: 17 us.
//
// Number ranges as in attention_prompt.cu: queries normalised per row by a
// power of two, value scales by that of the largest so far, the maximum
// followed lazily; fp32 splits queries and probabilities in two fp16 parts.
#include <float.h>

#include "attention_math.cuh"

namespace ndl {

namespace {

constexpr int kSplitStages = 2;
constexpr int kSplitCtas = 148;                       // one CTA an SM
constexpr int kWholePages = 16;                       // of a row: up to here a CTA takes an item, if they are few (above)
constexpr int kHeadBlock = 16;                        // query heads an item holds
constexpr uint32_t kSplitWait = 1u << 22;             // tests of about a microsecond: a few seconds
// A piece: per head 64 outputs, m and l (padded to 16 bytes).
constexpr int kPieceHead = 68;
constexpr int kJoinThreads = 256;

// Wide: 9 to 16 heads an item (both halves of the products' 16 rows).
template <bool kWide, bool kSplit>
struct SplitShape {
    // as many warps as their rings, pieces and probabilities leave room for in shared memory
    static constexpr int kWarps = kWide ? (kSplit ? 8 : 9) : (kSplit ? 10 : 11);
    static constexpr int kThreads = 32 * kWarps, kHeads = kWide ? 16 : 8;
};

// An item that reaches over a CTA's first record: where it is, and its records.
struct __align__(16) SplitItem {
    long long begin, end;
    int row, item;
};

struct SplitArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int32_t *row_slot, *row_len;
    int rows, heads, group, blocks, window;  // blocks: items a kv head and row
    int piece_heads;                         // heads a piece holds: min(group, 16)
    bool whole;                              // a CTA an item
    float scale;
    PagedCache c;
    SplitItem *over;  // [kSplitCtas + 1]: the item at a CTA's first record if it began before (else row -1); behind
                      // them, in `end`, the call's records
    float *pieces;    // [kSplitCtas][2][piece_heads][kPieceHead]
};

// Pages [first, last) that a row reads (none for an empty or a bad row).
__device__ __forceinline__ bool row_pages(const SplitArgs &a, int row, int &first, int &last) {
    const int slot = a.row_slot[row], len = a.row_len[row];
    first = last = 0;
    if (slot < 0 || slot >= a.c.slots || len < 0 || len > a.c.max_pages * kPagePositions) return false;
    if (len == 0) return true;
    first = (a.window ? max(0, len - a.window) : 0) / kPagePositions;
    last = (len - 1) / kPagePositions + 1;
    return true;
}
// 64-bit quotients are slow, and records hardly ever need them.
__device__ __forceinline__ long long quotient(long long a, int b) {
    return a >> 32 == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// `count` records in even shares: the first `more` workers take each + 1, the others each.
struct Shares {
    long long each;
    int more;
    __device__ __forceinline__ Shares(long long count, int workers) {
        each = quotient(count, workers);
        more = (int)(count - each * workers);
    }
    __device__ __forceinline__ long long start(int w) const { return each * w + min(w, more); }
    __device__ __forceinline__ int holder(long long record) const {
        const long long split = (each + 1) * more;
        return record < split ? (int)quotient(record, (int)(each + 1)) : more + (int)quotient(record - split, (int)each);
    }
};

// Where a worker stands: item (row, virtual head) and page of it.
struct SplitCursor {
    int row, item, page, first, last;
};

// Lane (g, t) = (lane / 4, lane % 4).  Products have positions (then dims) as
// their 16 rows and heads as their 8 columns, NB column blocks (1 or 2):
// a lane's scores and outputs are those of heads 8 b + 2 t and + 1, its query
// fragments those of head 8 b + g.
template <int NB>
struct SplitState {
    float o[NB][4][4];  // dims 16 D + g (two heads) and + 8
    float top[NB][2], total[NB][2];
    int exponent;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int d = 0; d < 4; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[b][d][i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; e++) top[b][e] = -INFINITY, total[b][e] = 0.0f;
        }
        exponent = kMinExponent;
    }
};

// The query fragments of an item: k-step s covers dims 16 s + 4 t .. + 3 (as the key fragments hold them).
template <int NB, bool kSplit>
struct SplitQuery {
    uint32_t b[kSplit ? 2 : 1][NB][4][2];  // [part][head block][k-step][dim pair]
    float factor[NB][2];                   // scores -> binary orders, of heads 8 b + 2 t and + 1
};

template <class T, int NB, bool kSplit>
__device__ __forceinline__ void load_query(const SplitArgs &a, int row, int item, int lane, SplitQuery<NB, kSplit> &q) {
    const int kv = item / a.blocks, block = item - kv * a.blocks;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int in_group = block * kHeadBlock + b * 8 + (lane >> 2);
        const bool there = in_group < a.group;
        const T *src = static_cast<const T *>(a.q) + (size_t)row * a.q_stride +
                       ((size_t)kv * a.group + (there ? in_group : 0)) * kHeadDim + (lane & 3) * 4;
        float x[4][4], peak = 0.0f;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            load4(src + 16 * s, x[s]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (!there) x[s][i] = 0.0f;
                peak = fmaxf(peak, fabsf(x[s][i]));
            }
        }
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
        float up, down;
        query_norm(peak, up, down);
        const float factor = fmaxf(down * a.scale * kLog2E, FLT_MIN);  // not zero: it multiplies infinities
#pragma unroll
        for (int e = 0; e < 2; e++) q.factor[b][e] = __shfl_sync(0xffffffffu, factor, (2 * (lane & 3) + e) * 4);
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const float f0 = x[s][2 * p] * up, f1 = x[s][2 * p + 1] * up;
                q.b[0][b][s][p] = half_pair(f0, f1);
                if constexpr (kSplit) q.b[kSplit ? 1 : 0][b][s][p] = half_rest(f0, f1, q.b[0][b][s][p]);
            }
    }
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Four 8x8 matrices of fp16, each stored transposed.
__device__ __forceinline__ void stmatrix4_trans(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2),
                 "r"(r3)
                 : "memory");
}

// The probabilities' place between the products: per head 64 positions of
// fp16, rows 16 bytes apart from a multiple of 128 (no bank conflicts).
constexpr int kProbRow = 2 * kPagePositions + 16;
template <int NB, bool kSplit>
constexpr int kProbBytes = (kSplit ? 2 : 1) * NB * 8 * kProbRow;

template <bool kWide, bool kSplit>
struct SplitSmem {
    using Sh = SplitShape<kWide, kSplit>;
    uint8_t ring[Sh::kWarps][kSplitStages][kKvBlockBytes];  // at the end, a warp's second piece
    float first[Sh::kWarps][Sh::kHeads * kPieceHead];       // a warp's first piece
    uint8_t prob[Sh::kWarps][kProbBytes<kWide ? 2 : 1, kSplit>];
    SplitItem info[Sh::kWarps][2];                          // the pieces' items (row -1: no piece)
    uint64_t full[Sh::kWarps][kSplitStages];
    long long sums[Sh::kThreads + 1];
    long long begin, end, records;                          // the CTA's records, and the call's
};
static_assert(kHeadBlock * kPieceHead * 4 <= kKvBlockBytes, "a piece fits a ring record");

// One page into the state.  Positions [from, upto) of it count.
template <int NB, bool kSplit>
__device__ __forceinline__ void attend_page(const uint8_t *rec, uint8_t *prob, int from, int upto, int lane,
                                            const SplitQuery<NB, kSplit> &q, SplitState<NB> &st) {
    constexpr int kParts = kSplit ? 2 : 1;
    const int g = lane >> 2, t = lane & 3;
    // scores of positions 16 T + g and + 8, heads 2 t and + 1
    float s[NB][4][4];
#pragma unroll
    for (int T = 0; T < 4; T++) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[b][T][i] = 0.0f;
        uint32_t x[2][8];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            // words: (row g, dims), (row g + 8, dims), then dims + 16
            const uint4 w = *reinterpret_cast<const uint4 *>(rec + T * 1024 + k * 512 + lane * 16);
            codes_to_half(w.x, x[k][0], x[k][1]);
            codes_to_half(w.y, x[k][2], x[k][3]);
            codes_to_half(w.z, x[k][4], x[k][5]);
            codes_to_half(w.w, x[k][6], x[k][7]);
        }
        // the small part first: the accumulator truncates what is added
#pragma unroll
        for (int part = kParts - 1; part >= 0; part--)
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    mma_16816(s[b][T], x[k][0], x[k][2], x[k][1], x[k][3], q.b[part][b][2 * k][0], q.b[part][b][2 * k][1]);
                    mma_16816(s[b][T], x[k][4], x[k][6], x[k][5], x[k][7], q.b[part][b][2 * k + 1][0], q.b[part][b][2 * k + 1][1]);
                }
    }
    // the positions' scales: keys (2 T + h) in a row, values over 2^exponent (of the largest so far) times 2^8
    const bool whole = from <= 0 && upto >= kPagePositions;
    float ks[8], vs[8];
    {
        const float4 *k4 = reinterpret_cast<const float4 *>(rec + kKScaleOffset) + 2 * g;
        const float4 k0 = k4[0], k1 = k4[1];
        ks[0] = k0.x, ks[1] = k0.y, ks[2] = k0.z, ks[3] = k0.w, ks[4] = k1.x, ks[5] = k1.y, ks[6] = k1.z, ks[7] = k1.w;
    }
    int big = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int p = 8 * i + g;
        vs[i] = reinterpret_cast<const float *>(rec + kVScaleOffset)[p];
        if (!whole && (p < from || p >= upto)) vs[i] = 0.0f;
        big = max(big, scale_exponent(vs[i]));
    }
    const int exponent = max(st.exponent, __reduce_max_sync(0xffffffffu, big) - 126);
    const float norm = pow2(8 - exponent);
    const float shrink = exponent > st.exponent ? exp2_approx((float)(st.exponent - exponent)) : 1.0f;
    st.exponent = exponent;
#pragma unroll
    for (int i = 0; i < 8; i++) vs[i] *= norm;
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float peak[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 8; i++) {  // position 8 i + g
            const int p = 8 * i + g;
            float &x0 = s[b][i >> 1][2 * (i & 1)], &x1 = s[b][i >> 1][2 * (i & 1) + 1];
            x0 *= ks[i], x1 *= ks[i];
            if (!whole && (p < from || p >= upto)) x0 = x1 = -INFINITY;
            peak[0] = fmaxf(peak[0], x0), peak[1] = fmaxf(peak[1], x1);
        }
        float keep[2], base[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) peak[e] = fmaxf(peak[e], __shfl_xor_sync(0xffffffffu, peak[e], o));
            keep[e] = shrink;
            float &top = st.top[b][e];
            if ((peak[e] - top) * q.factor[b][e] > kLazy || (top == -INFINITY && peak[e] > -INFINITY)) {
                const float k = top == -INFINITY ? 0.0f : exp2_approx((top - peak[e]) * q.factor[b][e]);
                st.total[b][e] *= k, keep[e] *= k;
                top = peak[e];
            }
            base[e] = top == -INFINITY ? 0.0f : top * q.factor[b][e];
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
            for (int d = 0; d < 4; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) st.o[b][d][i] *= keep[i & 1];
        }
        // probabilities, stored transposed: a row of heads, 8 positions a matrix
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float e0 = exp2_approx(fmaf(s[b][i >> 1][2 * (i & 1)], q.factor[b][0], -base[0]));
            const float e1 = exp2_approx(fmaf(s[b][i >> 1][2 * (i & 1) + 1], q.factor[b][1], -base[1]));
            st.total[b][0] += e0, st.total[b][1] += e1;
            const float p0 = e0 * vs[i], p1 = e1 * vs[i];
            hi[i] = half_pair(p0, p1);
            if constexpr (kSplit) lo[i] = half_rest(p0, p1, hi[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            // lane 8 m + r gives the address of matrix m's row r (head r): positions 8 (i + m) ..
            const uint32_t at = smem_u32(prob) + (b * 8 + (lane & 7)) * kProbRow + (i + (lane >> 3)) * 16;
            stmatrix4_trans(at, hi[i], hi[i + 1], hi[i + 2], hi[i + 3]);
            if constexpr (kSplit) stmatrix4_trans(at + NB * 8 * kProbRow, lo[i], lo[i + 1], lo[i + 2], lo[i + 3]);
        }
    }
    __syncwarp();
    // O += V P: dims as rows; k-step T covers positions 16 T + 4 t .. + 3 of lane t, as ldmatrix hands the codes out
    uint2 p[kParts][NB][4];
#pragma unroll
    for (int part = 0; part < kParts; part++)
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int T = 0; T < 4; T++)
                p[part][b][T] = *reinterpret_cast<const uint2 *>(prob + ((part * NB + b) * 8 + g) * kProbRow + (16 * T + 4 * t) * 2);
#pragma unroll
    for (int D = 0; D < 4; D++) {
        // (fp32: the parts of a page by themselves, then into the output by additions that round)
        float part_o[kParts][NB][4];
        if constexpr (kSplit) {
#pragma unroll
            for (int i = 0; i < kParts * NB * 4; i++) (&part_o[0][0][0])[i] = 0.0f;
        }
#pragma unroll
        for (int T = 0; T < 4; T += 2) {
            // matrices: dims 16 D + 0..7 and + 8..15 of chunk T, then of chunk T + 1
            const int d = 16 * D + (lane >> 3 & 1) * 8 + (lane & 7), c = T + (lane >> 4);
            uint32_t w[4];
            ldmatrix4(w, smem_u32(rec + kVOffset + d * 64 + ((c ^ ((d >> 1) & 3)) << 4)));
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t x[4];
                codes_to_half(w[2 * u], x[0], x[1]);
                codes_to_half(w[2 * u + 1], x[2], x[3]);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int part = 0; part < kParts; part++)
                        mma_16816(kSplit ? part_o[part][b] : st.o[b][D], x[0], x[2], x[1], x[3], p[part][b][T + u].x,
                                  p[part][b][T + u].y);
            }
        }
        if constexpr (kSplit) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) st.o[b][D][i] += part_o[kParts - 1][b][i] + part_o[0][b][i];
        }
    }
    __syncwarp();  // the probabilities' place is free again
}

// A piece joined into the running (top, sum, o0, o1) of a lane's two dims.
struct SplitJoin {
    float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    __device__ __forceinline__ void add(float2 ml, float2 v) {
        const float m = fmaxf(top, ml.x);
        const float keep = top == m ? 1.0f : exp2f(top - m), f = ml.x == m ? ml.y : ml.y * exp2f(ml.x - m);
        sum = fmaf(sum, keep, f), o0 = fmaf(o0, keep, f * v.x), o1 = fmaf(o1, keep, f * v.y);
        top = m;
    }
};

template <class T, bool kWide>
__global__ void __launch_bounds__(SplitShape<kWide, sizeof(T) == 4>::kThreads, 1) attention_split_kernel(SplitArgs a) {
    constexpr bool kSplit = sizeof(T) == 4;
    constexpr int NB = kWide ? 2 : 1, kWarps = SplitShape<kWide, kSplit>::kWarps, kThreads = 32 * kWarps;
    extern __shared__ uint8_t smem_raw[];
    using Smem = SplitSmem<kWide, kSplit>;
    Smem &s = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int virtual_heads = a.c.heads * a.blocks;
    pdl_trigger();  // the joining kernel waits for this one's end by itself

    if (lane < kSplitStages) mbar_init(&s.full[warp][lane], 1);
    if (lane < 2) s.info[warp][lane].row = -1;
    fence_mbar_init();
    __syncwarp();
    SplitCursor cur;
    long long records = 0, cta_begin = 0, cta_end, begin, end;  // the call's records; of them the CTA's, and this warp's
    long long item_at = 0;                                      // record index of the current item's first page
    int len = 0;
    if (a.whole) {  // a CTA an item, whose records count from 0
        cur.row = blockIdx.x / virtual_heads, cur.item = blockIdx.x - cur.row * virtual_heads;
        row_pages(a, cur.row, cur.first, cur.last);
        cta_end = cur.last - cur.first;
        const Shares of_warps(cta_end, kWarps);
        begin = of_warps.start(warp), end = of_warps.start(warp + 1);
        cur.page = cur.first + (int)begin;
        len = a.row_len[cur.row];
    } else {
        // Records before each row.  Up to 32 rows: every warp scans them by itself, lane = row.  More: a thread sums a
        // run of rows, the CTA scans the runs.
        const auto row_records = [&](int row) {
            int first, last;
            row_pages(a, row, first, last);
            return (long long)(last - first) * virtual_heads;
        };
        const auto scan = [&](long long x) {  // over the warp, this lane included
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += up;
            }
            return x;
        };
        long long at = 0;  // records before the first one's row
        long long upto = 0, mine = 0;
        if (a.rows <= 32) {
            mine = lane < a.rows ? row_records(lane) : 0, upto = scan(mine);
            records = __shfl_sync(0xffffffffu, upto, 31);
        } else {
            const int run = (a.rows + kThreads - 1) / kThreads;
            for (int i = threadIdx.x * run; i < min(a.rows, (int)(threadIdx.x + 1) * run); i++) mine += row_records(i);
            const long long sum = scan(mine);
            if (lane == 31) s.sums[warp + 1] = sum;
            __syncthreads();
            long long before = sum;
            for (int w = 0; w < warp; w++) before += s.sums[w + 1];
            __syncthreads();
            s.sums[threadIdx.x + 1] = before;
            if (threadIdx.x == 0) s.sums[0] = 0;
            __syncthreads();
            records = s.sums[kThreads];
        }
        const Shares of_ctas(records, gridDim.x);
        cta_begin = of_ctas.start(blockIdx.x), cta_end = of_ctas.start(blockIdx.x + 1);
        const Shares of_warps(cta_end - cta_begin, kWarps);
        begin = cta_begin + of_warps.start(warp), end = cta_begin + of_warps.start(warp + 1);
        if (begin < end) {
            if (a.rows <= 32) {
                cur.row = __ffs(__ballot_sync(0xffffffffu, upto > begin)) - 1;
                at = __shfl_sync(0xffffffffu, upto - mine, cur.row);
            } else {
                const int run = (a.rows + kThreads - 1) / kThreads;
                int lo = 0, hi = kThreads;  // the run: sums[lo] <= begin < sums[hi]
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s.sums[mid] <= begin) lo = mid;
                    else hi = mid;
                }
                at = s.sums[lo];
                for (cur.row = lo * run;; cur.row++) {
                    const long long n = row_records(cur.row);
                    if (begin < at + n) break;
                    at += n;
                }
            }
            row_pages(a, cur.row, cur.first, cur.last);
            const int pages = cur.last - cur.first;
            cur.item = (int)quotient(begin - at, pages);
            item_at = at + (long long)cur.item * pages;
            cur.page = cur.first + (int)(begin - item_at);
            len = a.row_len[cur.row];
        }
    }

    if (threadIdx.x == 0) s.begin = cta_begin, s.end = cta_end, s.records = records;  // for the end

    // the copies' own place, ahead of the reading
    SplitCursor ahead = cur;
    int ids = -1, ids_row = -1, ids_at = -1, slot = 0;
    uint32_t bad = 0;  // ring stages whose page is missing
    long long next = begin;
    auto issue = [&](int stage) {  // the copy of record `next`
        const int at = ahead.page & ~31;
        if (ahead.row != ids_row || at != ids_at) {
            ids_row = ahead.row, ids_at = at;
            slot = a.row_slot[ahead.row];
            ids = at + lane < ahead.last ? cache_page(a.c, slot, at + lane) : -1;
        }
        const int page = __shfl_sync(0xffffffffu, ids, ahead.page & 31);
        bad = page < 0 ? bad | (1u << stage) : bad & ~(1u << stage);
        if (page >= 0 && lane == 0) {
            mbar_arrive_expect_tx(&s.full[warp][stage], kKvBlockBytes);
            bulk_g2s(s.ring[warp][stage], cache_record(a.c, page, ahead.item / a.blocks), kKvBlockBytes,
                     &s.full[warp][stage]);
        }
        next++;
        if (++ahead.page == ahead.last && next < end) {
            if (++ahead.item == virtual_heads) {
                ahead.item = 0;
                do {
                    ahead.row++;
                    row_pages(a, ahead.row, ahead.first, ahead.last);
                } while (ahead.first == ahead.last);
            }
            ahead.page = ahead.first;
        }
    };
    for (int i = 0; i < kSplitStages && next < end; i++) issue(i);

    SplitQuery<NB, kSplit> q;
    SplitState<NB> st;
    if (begin < end) load_query<T, NB, kSplit>(a, cur.row, cur.item, lane, q);
    st.clear();
    int piece = 0;           // this warp's pieces: 0 starts at its first record, 1 is a later one
    uint32_t phases = 0;     // parity of each stage's next completed copy
    bool timed_out = false;
    int stage = 0;
    for (long long rec = begin; rec < end; rec++) {
        if (bad >> stage & 1) {
#pragma unroll
            for (int b = 0; b < NB; b++) st.total[b][0] = st.total[b][1] = __int_as_float(0x7fc00000);
            if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        } else {
            const bool ok = mbar_wait_bounded(&s.full[warp][stage], phases >> stage & 1, kSplitWait);
            if (!__all_sync(0xffffffffu, ok)) {
                timed_out = true;
                break;
            }
            phases ^= 1u << stage;
            const int at = cur.page * kPagePositions;
            attend_page<NB, kSplit>(s.ring[warp][stage], s.prob[warp], a.window ? len - a.window - at : 0, len - at, lane, q, st);
        }
        __syncwarp();
        if (next < end) issue(stage);
        stage = stage + 1 == kSplitStages ? 0 : stage + 1;

        const bool item_ends = cur.page + 1 == cur.last;
        if (item_ends || rec + 1 == end) {
            // the item, or this warp's piece of it
            const bool alone = item_ends && item_at >= begin;
            const int kv = cur.item / a.blocks, block = cur.item - kv * a.blocks;
            const float back = pow2(st.exponent - 8);
            // outputs through shared memory, [head][dim]: a piece to its place, an item by 16 dims at a time
            float *place = piece ? reinterpret_cast<float *>(s.ring[warp][0]) : s.first[warp];
            float *stage16 = reinterpret_cast<float *>(s.prob[warp]);
            const int heads = min(kHeadBlock, a.group - block * kHeadBlock);
            T *dst = static_cast<T *>(a.out) + (size_t)cur.row * a.out_stride +
                     ((size_t)kv * a.group + block * kHeadBlock) * kHeadDim;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float &total = st.total[b][e];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                    const float f = 1.0f / total;
#pragma unroll
                    for (int d = 0; d < 4; d++) st.o[b][d][e] *= f, st.o[b][d][2 + e] *= f;
                }
#pragma unroll
            for (int d = 0; d < 4; d++) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int head = b * 8 + 2 * (lane & 3) + (i & 1), dim = (lane >> 2) + 8 * (i >> 1);
                        const float x = st.o[b][d][i] * back;
                        if (alone) stage16[head * 16 + dim] = x;
                        else if (head < heads) place[head * kPieceHead + 16 * d + dim] = x;
                    }
                if (alone) {
                    __syncwarp();
                    for (int i = lane; i < heads * 8; i += 32) {
                        const float2 v = *reinterpret_cast<const float2 *>(stage16 + 2 * i);
                        store2(dst + (i >> 3) * kHeadDim + 16 * d + 2 * (i & 7), v.x, v.y);
                    }
                    __syncwarp();
                }
            }
            if (!alone && (lane >> 2) == 0) {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int head = b * 8 + 2 * lane + e;
                        if (head < heads)
                            *reinterpret_cast<float2 *>(place + head * kPieceHead + kHeadDim) =
                                make_float2(st.top[b][e] * q.factor[b][e], st.total[b][e]);
                    }
            }
            if (!alone && lane == 0) s.info[warp][piece] = SplitItem{item_at, item_at + (cur.last - cur.first), cur.row, cur.item};
            if (rec + 1 < end) {
                item_at = rec + 1;
                piece = 1;
                if (++cur.item == virtual_heads) {
                    cur.item = 0;
                    do {
                        cur.row++;
                        row_pages(a, cur.row, cur.first, cur.last);
                    } while (cur.first == cur.last);
                    len = a.row_len[cur.row];
                }
                cur.page = cur.first;
                load_query<T, NB, kSplit>(a, cur.row, cur.item, lane, q);
                st.clear();
            }
        } else {
            cur.page++;
        }
    }
    if (timed_out) {
        if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusTimeout);
        // every copy in flight lands before the warp exits (bounded)
        for (int i = 0; i < kSplitStages; i++)
            if (!(bad >> i & 1)) mbar_wait_bounded(&s.full[warp][i], phases >> i & 1, kSplitWait);
    }
    if (!a.whole && threadIdx.x == 0) {
        a.over[blockIdx.x].row = -1;
        if (blockIdx.x == 0) a.over[kSplitCtas].end = s.records;
    }
    __syncthreads();

    // The pieces: each item's first warp here joins what the warps behind it hold of it.
#pragma unroll 1
    for (int slot = 0; slot < 2; slot++) {
        const SplitItem it = s.info[warp][slot];
        if (it.row < 0 || (slot == 0 && warp > 0 && it.begin < begin)) continue;
        int last = warp;
        while (last + 1 < kWarps && s.info[last + 1][0].row >= 0 && s.info[last + 1][0].begin == it.begin) last++;
        const bool whole = it.begin >= s.begin && it.end <= s.end;
        const int kv = it.item / a.blocks, block = it.item - kv * a.blocks;
        const int heads = min(kHeadBlock, a.group - block * kHeadBlock);
        for (int h = 0; h < heads; h++) {
            SplitJoin j;
            for (int w = warp; w <= last; w++) {
                const float *p = (w == warp && slot ? reinterpret_cast<const float *>(s.ring[w][0]) : s.first[w]) + h * kPieceHead;
                j.add(*reinterpret_cast<const float2 *>(p + kHeadDim), *reinterpret_cast<const float2 *>(p + 2 * lane));
            }
            if (whole) {
                store2(static_cast<T *>(a.out) + (size_t)it.row * a.out_stride +
                           ((size_t)kv * a.group + block * kHeadBlock + h) * kHeadDim + 2 * lane,
                       j.o0 / j.sum, j.o1 / j.sum);
            } else {
                float *dst = a.pieces + (((size_t)blockIdx.x * 2 + (it.begin > s.begin)) * a.piece_heads + h) * kPieceHead;
                *reinterpret_cast<float2 *>(dst + 2 * lane) = make_float2(j.o0 / j.sum, j.o1 / j.sum);
                if (lane == 0) *reinterpret_cast<float2 *>(dst + kHeadDim) = make_float2(j.top, j.sum);
            }
        }
        if (!whole && it.begin < s.begin && lane == 0) a.over[blockIdx.x] = it;
    }
    // rows that read nothing
    for (int row = blockIdx.x * kWarps + warp; row < a.rows; row += gridDim.x * kWarps) {
        int first, last;
        const bool good = row_pages(a, row, first, last);
        if (first < last) continue;
        if (!good && lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        T *dst = static_cast<T *>(a.out) + (size_t)row * a.out_stride;
        const T value = from_float<T>(good ? 0.0f : __int_as_float(0x7fc00000));
        for (int i = lane; i < a.heads * kHeadDim; i += 32) dst[i] = value;
    }
}

// Joins the pieces of an item that several CTAs hold, in order:
//   out = sum w_i o_i / sum w_i,  w_i = l_i 2^(m_i - max m)
// A CTA takes one head of the item at the start of split CTA blockIdx.x + 1,
// if that is the first start inside the item; its warps share out the pieces,
// whose loads go out in batches.
template <class T>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(SplitArgs a, int ctas) {
    constexpr int kWarps = kJoinThreads / 32, kBatch = 8;
    __shared__ float acc[kWarps][kHeadDim];
    __shared__ float2 part_ml[kWarps];
    const int cta = blockIdx.x + 1, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const SplitItem it = a.over[cta];
    if (it.row < 0) return;
    const Shares shares(a.over[kSplitCtas].end, ctas);
    const int block = it.item % a.blocks, kv = it.item / a.blocks;
    const int w0 = shares.holder(it.begin), w1 = shares.holder(it.end - 1);
    if (w0 != cta - 1 || block * kHeadBlock + h >= a.group) return;
    const int first_slot = it.begin > shares.start(w0);  // its first CTA's second piece, unless it began with that CTA
    const int count = w1 - w0 + 1, per = (count + kWarps - 1) / kWarps;
    const int from = w0 + warp * per, to = min(w1 + 1, from + per);
    SplitJoin j;
    for (int base = from; base < to; base += kBatch) {
        float2 ml[kBatch], v[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int w = min(base + i, to - 1);
            const float *p = a.pieces + (((size_t)w * 2 + (w == w0 ? first_slot : 0)) * a.piece_heads + h) * kPieceHead;
            ml[i] = *reinterpret_cast<const float2 *>(p + kHeadDim);
            v[i] = *reinterpret_cast<const float2 *>(p + 2 * lane);
        }
#pragma unroll
        for (int i = 0; i < kBatch; i++)
            if (base + i < to) j.add(ml[i], v[i]);
    }
    *reinterpret_cast<float2 *>(&acc[warp][2 * lane]) = make_float2(j.o0, j.o1);
    if (lane == 0) part_ml[warp] = make_float2(j.top, j.sum);
    __syncthreads();
    if (warp != 0) return;
    float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int i = 0; i < kWarps; i++) m = fmaxf(m, part_ml[i].x);
    for (int i = 0; i < kWarps; i++) {
        if (w0 + i * per > w1) break;  // no pieces from here on
        const float f = part_ml[i].x == m ? 1.0f : exp2f(part_ml[i].x - m);
        sum += part_ml[i].y * f, o0 += acc[i][2 * lane] * f, o1 += acc[i][2 * lane + 1] * f;
    }
    store2(static_cast<T *>(a.out) + (size_t)it.row * a.out_stride + ((size_t)kv * a.group + block * kHeadBlock + h) * kHeadDim +
               2 * lane,
           o0 / sum, o1 / sum);
}

}  // namespace

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

constexpr size_t kOverBytes = (kSplitCtas + 1) * sizeof(SplitItem);

}  // namespace ndl

using namespace ndl;

// The items over the CTAs' starts, and two pieces a CTA.
extern "C" NDL_API size_t ndl_attention_split_workspace(int rows, int heads, int kv_heads, int max_pages) {
    if (rows <= 0 || heads <= 0 || kv_heads <= 0 || max_pages <= 0 || heads % kv_heads != 0) return 0;
    const int held = heads / kv_heads < kHeadBlock ? heads / kv_heads : kHeadBlock;
    return kOverBytes + (size_t)kSplitCtas * 2 * held * kPieceHead * sizeof(float);
}

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
    NDL_REQUIRE(aligned(workspace, 16) && workspace && workspace_bytes >= need, "workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
    const int group = heads / kv_heads;
    const int blocks = (group + kHeadBlock - 1) / kHeadBlock;
    const int pages = window && window / kPagePositions + 2 < max_pages ? window / kPagePositions + 2 : max_pages;
    const long long items = (long long)rows * kv_heads * blocks;
    const bool whole = pages <= kWholePages && items <= kSplitCtas;
    SplitArgs a{q, out, q_stride, out_stride, row_slot, row_len, rows, heads, group,
                blocks, window, group < kHeadBlock ? group : kHeadBlock, whole, scale,
                {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                 kv_heads, status},
                static_cast<SplitItem *>(workspace),
                reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kOverBytes)};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const bool wide = group > 8;
        const auto kernel = wide ? attention_split_kernel<T, true> : attention_split_kernel<T, false>;
        using Wide = SplitSmem<true, sizeof(T) == 4>;
        using Narrow = SplitSmem<false, sizeof(T) == 4>;
        static_assert(sizeof(Wide) + 128 <= 232448 && sizeof(Narrow) + 128 <= 232448, "shared memory of an SM");
        const size_t smem = (wide ? sizeof(Wide) : sizeof(Narrow)) + 128;
        static DeviceOnce attribute;  // the attributes belong to the kernels on one device
        const int st = attribute.run([&] {
            cudaError_t e = cudaFuncSetAttribute(attention_split_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)sizeof(Wide) + 128);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(attention_split_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)sizeof(Narrow) + 128);
            return e == cudaSuccess ? (int)NDL_OK
                                    : set_error(NDL_ERR_CUDA, "split attention smem: %s", cudaGetErrorString(e));
        });
        if (st != NDL_OK) return st;
        const int threads = wide ? SplitShape<true, sizeof(T) == 4>::kThreads : SplitShape<false, sizeof(T) == 4>::kThreads;
        kernel<<<whole ? (unsigned)items : kSplitCtas, threads, smem, (cudaStream_t)stream>>>(a);
        const int rc2 = check_launch("attention_split");
        if (rc2 != NDL_OK || whole) return rc2;
        PdlScope early(true);  // the join's launch overlaps the kernel above; it waits for its end before reading
        launch_kernel(attention_join_kernel<T>, dim3(kSplitCtas - 1, a.piece_heads), dim3(kJoinThreads), 0,
                      (cudaStream_t)stream, a, kSplitCtas);
        return check_launch("attention_join");
    });
}
