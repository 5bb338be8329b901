// Attention of single tokens over the paged int8 cache, split over its length.
//
// A row's query heads that share a kv head (at most 16 at a time) attend
// together; such an item reads one 8704-byte record per page.  All records of
// a call, item after item, are dealt out evenly: worker w of W (a warp) takes
// its share in order, T / W of them or one more, whatever the rows' lengths are, so one
// long row fills the card as well as many ragged ones.  A worker streams its
// records through its own ring in shared memory (one bulk copy each, 12 warps
// x 2 records = 209 KB in flight an SM against the ~45 KB that bandwidth times
// latency asks for; 8 warps x 3 took 239 us where these take 222) and keeps a running maximum, sum and output per head:
//   S = Q K^T, O += (e vs) V   mma.sync m16n8k16 (heads x positions / dims);
// the codes become fp16 exactly in registers, from the fragments the pages
// hold.  Tensor cores because a position costs 128 products a head and 128
// conversions, and a kv head's group shares the conversions; tcgen05 would
// need tiles of 128 rows, and there are at most 16.
// An item inside one worker is finished there; pieces of the others (O / l,
// m, l) go to the workspace, and a second kernel, launched early, joins them
// in order, so the result does not depend on timing.
//
// Number ranges as in attention_prompt.cu: queries normalised per row by a
// power of two, value scales by that of the largest so far, the maximum
// followed lazily; fp32 splits queries and probabilities in two fp16 parts.
#include <float.h>

#include "attention_math.cuh"

namespace ndl {

namespace {

constexpr int kSplitWarps = 12, kSplitThreads = 32 * kSplitWarps, kSplitStages = 2;
constexpr int kSplitCtas = 148;                       // one CTA an SM
constexpr int kSplitWorkers = kSplitCtas * kSplitWarps;
constexpr int kHeadBlock = 16;                        // query heads an item holds
constexpr uint32_t kSplitWait = 1u << 22;             // tests of about a microsecond: a few seconds
// A piece: per head 64 outputs, m and l (padded to 16 bytes).
constexpr int kPieceHead = 68;
constexpr int kJoinThreads = 256;
constexpr int kJoinItems = 592;                       // items from which a CTA joins all heads of one

struct SplitArgs {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const int32_t *row_slot, *row_len;
    int rows, heads, group, blocks, window;  // blocks: items a kv head and row
    int piece_heads;                         // heads a piece holds: min(group, 16)
    float scale;
    PagedCache c;
    long long *prefix;  // [rows + 1]: records before each row
    float *pieces;      // [kSplitWorkers][2][piece_heads][kPieceHead]
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
// The records' shares: workers 0 .. more - 1 take each + 1, the others each.
struct Shares {
    long long each;
    int workers, more;
    __device__ __forceinline__ explicit Shares(long long records) {
        workers = records < kSplitWorkers ? (int)records : kSplitWorkers;
        each = workers ? quotient(records, workers) : 0;
        more = (int)(records - each * workers);
    }
    __device__ __forceinline__ long long start(int w) const { return each * w + min(w, more); }
    __device__ __forceinline__ int holder(long long record) const {
        const long long split = (each + 1) * more;
        return record < split ? (int)quotient(record, (int)(each + 1)) : more + (int)quotient(record - split, (int)each);
    }
};

struct SplitSmem {
    uint8_t ring[kSplitWarps][kSplitStages][kKvBlockBytes];
    uint64_t full[kSplitWarps][kSplitStages];
    long long sums[kSplitThreads + 1];
};

// Where a worker stands: item (row, virtual head) and page of it.
struct SplitCursor {
    int row, item, page, first, last;
};

// The state of one item's heads: outputs (8 dim blocks), maximum, sum.
template <bool kWide>
struct SplitState {
    static constexpr int kRows = kWide ? 2 : 1;  // heads lane / 4 and, wide, lane / 4 + 8
    float o[8][4];
    float top[kRows], total[kRows];
    int exponent;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < 8; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[d][i] = 0.0f;
#pragma unroll
        for (int r = 0; r < kRows; r++) top[r] = -INFINITY, total[r] = 0.0f;
        exponent = kMinExponent;
    }
};

// The query fragments of an item: k-step (s, h) covers dims 32 s + 16 h + 4 t
// .. + 3 of lane t = lane & 3 (as the key fragments hold them).
template <bool kWide, bool kSplit>
struct SplitQuery {
    static constexpr int kRows = kWide ? 2 : 1;
    uint32_t a[kSplit ? 2 : 1][4][kRows][2];  // [part][k-step][head half][dim pair]
    float factor[kRows];                      // scores -> binary orders
};

template <class T, bool kWide, bool kSplit>
__device__ __forceinline__ void load_query(const SplitArgs &a, int row, int item, int lane,
                                           SplitQuery<kWide, kSplit> &q) {
    const int kv = item / a.blocks, block = item - kv * a.blocks;
#pragma unroll
    for (int r = 0; r < (kWide ? 2 : 1); r++) {
        const int in_group = block * kHeadBlock + r * 8 + (lane >> 2);
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
        q.factor[r] = fmaxf(down * a.scale * kLog2E, FLT_MIN);  // not zero: it multiplies infinities
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                const float f0 = x[s][2 * p] * up, f1 = x[s][2 * p + 1] * up;
                q.a[0][s][r][p] = half_pair(f0, f1);
                if constexpr (kSplit) q.a[kSplit ? 1 : 0][s][r][p] = half_rest(f0, f1, q.a[0][s][r][p]);
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

// One page into the state.  Positions [from, upto) of it count.
template <bool kWide, bool kSplit>
__device__ __forceinline__ void attend_page(const uint8_t *rec, int from, int upto, int lane,
                                            const SplitQuery<kWide, kSplit> &q, SplitState<kWide> &st) {
    constexpr int R = kWide ? 2 : 1;
    const int t = lane & 3;
    // scores: n-tile (T, h) holds positions 16 T + 8 h + 0..7, this lane's 2 t and 2 t + 1
    float s[4][2][4];
#pragma unroll
    for (int T = 0; T < 4; T++) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[T][h][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint4 w = *reinterpret_cast<const uint4 *>(rec + T * 1024 + k * 512 + lane * 16);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};  // (row, dims), (row + 8, dims), dims + 16 likewise
#pragma unroll
            for (int u = 0; u < 4; u++) {
                uint32_t b0, b1;
                codes_to_half(words[u], b0, b1);
                const int ks = 2 * k + (u >> 1);
#pragma unroll
                for (int part = 0; part < (kSplit ? 2 : 1); part++)
                    mma_16816(s[T][u & 1], q.a[part][ks][0][0], kWide ? q.a[part][ks][R - 1][0] : 0u,
                              q.a[part][ks][0][1], kWide ? q.a[part][ks][R - 1][1] : 0u, b0, b1);
            }
        }
    }
    // key scales of positions 2 t + e: eight (T, h) in a row
    const float4 *ks = reinterpret_cast<const float4 *>(rec + kKScaleOffset) + 4 * t;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float4 c0 = ks[2 * e], c1 = ks[2 * e + 1];
        const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
        for (int T = 0; T < 4; T++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < R; r++) s[T][h][2 * r + e] *= c[2 * T + h];
    }
    const bool whole = from <= 0 && upto >= kPagePositions;
    if (!whole) {
#pragma unroll
        for (int T = 0; T < 4; T++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int p = 16 * T + 8 * h + 2 * t + e;
                    if (p < from || p >= upto)
#pragma unroll
                        for (int r = 0; r < R; r++) s[T][h][2 * r + e] = -INFINITY;
                }
    }
    // value scales over 2^exponent (of the largest so far) times 2^8
    float2 vs[4][2];
    int big = 0;
#pragma unroll
    for (int T = 0; T < 4; T++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float2 v = *reinterpret_cast<const float2 *>(rec + kVScaleOffset + (16 * T + 8 * h + 2 * t) * 4);
            if (!whole) {
                const int p = 16 * T + 8 * h + 2 * t;
                if (p < from || p >= upto) v.x = 0.0f;
                if (p + 1 < from || p + 1 >= upto) v.y = 0.0f;
            }
            vs[T][h] = v;
            big = max(big, max(scale_exponent(v.x), scale_exponent(v.y)));
        }
    const int exponent = max(st.exponent, __reduce_max_sync(0xffffffffu, big) - 126);
    const float norm = pow2(8 - exponent);
    float keep[R], base[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        float peak = -INFINITY;
#pragma unroll
        for (int T = 0; T < 4; T++)
#pragma unroll
            for (int h = 0; h < 2; h++) peak = fmaxf(peak, fmaxf(s[T][h][2 * r], s[T][h][2 * r + 1]));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
        keep[r] = exponent > st.exponent ? exp2_approx((float)(st.exponent - exponent)) : 1.0f;
        if ((peak - st.top[r]) * q.factor[r] > kLazy || (st.top[r] == -INFINITY && peak > -INFINITY)) {
            const float k = st.top[r] == -INFINITY ? 0.0f : exp2_approx((st.top[r] - peak) * q.factor[r]);
            st.total[r] *= k, keep[r] *= k;
            st.top[r] = peak;
        }
        base[r] = st.top[r] == -INFINITY ? 0.0f : st.top[r] * q.factor[r];
    }
    st.exponent = exponent;
    bool moved = keep[0] != 1.0f;
    if constexpr (kWide) moved = moved || keep[R - 1] != 1.0f;
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int d = 0; d < 8; d++)
#pragma unroll
            for (int r = 0; r < R; r++) st.o[d][2 * r] *= keep[r], st.o[d][2 * r + 1] *= keep[r];
    }
    // probabilities: the second product's k-step T wants positions 4 t .. 4 t + 3 of 16 in lane t (as ldmatrix hands
    // out the value bytes), the scores left 2 t, 2 t + 1 and 8 + 2 t, 9 + 2 t there
    uint32_t p[kSplit ? 2 : 1][4][R][2];
    const int src = (lane & ~3) | ((2 * t) & 3);
#pragma unroll
    for (int r = 0; r < R; r++) {
        float sum = 0.0f;
#pragma unroll
        for (int T = 0; T < 4; T++) {
            uint32_t hi[2], lo[2] = {0, 0};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float e0 = exp2_approx(fmaf(s[T][h][2 * r], q.factor[r], -base[r]));
                const float e1 = exp2_approx(fmaf(s[T][h][2 * r + 1], q.factor[r], -base[r]));
                sum += e0 + e1;
                float p0 = e0 * (vs[T][h].x * norm), p1 = e1 * (vs[T][h].y * norm);
                hi[h] = half_pair(p0, p1);
                if constexpr (kSplit) lo[h] = half_rest(p0, p1, hi[h]);
            }
#pragma unroll
            for (int part = 0; part < (kSplit ? 2 : 1); part++) {
                const uint32_t *x = part ? lo : hi;
                const uint32_t a0 = __shfl_sync(0xffffffffu, x[0], src), b0 = __shfl_sync(0xffffffffu, x[1], src);
                const uint32_t a1 = __shfl_sync(0xffffffffu, x[0], src + 1);
                const uint32_t b1 = __shfl_sync(0xffffffffu, x[1], src + 1);
                p[part][T][r][0] = t < 2 ? a0 : b0;
                p[part][T][r][1] = t < 2 ? a1 : b1;
            }
        }
        st.total[r] += sum;
    }
    // O += P V: dims 8 D + (lane >> 2)
    const int d8 = lane & 7, T4 = lane >> 3;
#pragma unroll
    for (int D = 0; D < 8; D++) {
        const int d = 8 * D + d8;
        uint32_t w[4];
        ldmatrix4(w, smem_u32(rec + kVOffset + d * 64 + ((T4 ^ ((d >> 1) & 3)) << 4)));
#pragma unroll
        for (int T = 0; T < 4; T++) {
            uint32_t b0, b1;
            codes_to_half(w[T], b0, b1);
#pragma unroll
            for (int part = 0; part < (kSplit ? 2 : 1); part++)
                mma_16816(st.o[D], p[part][T][0][0], kWide ? p[part][T][R - 1][0] : 0u, p[part][T][0][1],
                          kWide ? p[part][T][R - 1][1] : 0u, b0, b1);
        }
    }
}

template <class T, bool kWide>
__global__ void __launch_bounds__(kSplitThreads, 1) attention_split_kernel(SplitArgs a) {
    constexpr bool kSplit = sizeof(T) == 4;
    constexpr int R = kWide ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    SplitSmem &s = *reinterpret_cast<SplitSmem *>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int virtual_heads = a.c.heads * a.blocks;
    pdl_trigger();  // the joining kernel waits for this one's end by itself

    for (int i = lane; i < kSplitStages; i += 32) mbar_init(&s.full[warp][i], 1);
    fence_mbar_init();
    __syncwarp();
    // Records before each row.  Up to 32 rows: every warp scans them by itself, lane = row.  More: a thread sums a run
    // of rows, the CTA scans the runs.
    const int worker = warp * gridDim.x + blockIdx.x;  // the first workers sit on different SMs
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
    SplitCursor cur;
    long long records, at;  // at: records before the first one's row
    const bool few = a.rows <= 32;
    const int run = (a.rows + kSplitThreads - 1) / kSplitThreads;
    if (few) {
        const long long mine = lane < a.rows ? row_records(lane) : 0, upto = scan(mine);
        records = __shfl_sync(0xffffffffu, upto, 31);
        if (blockIdx.x == 0 && warp == 0 && lane <= a.rows) {
            a.prefix[lane] = upto - mine;
            if (lane == 31) a.prefix[a.rows] = upto;  // 32 rows: one entry more than lanes
        }
        const Shares shares(records);
        if (worker >= shares.workers) return;
        const long long begin = shares.start(worker);
        const int l = __ffs(__ballot_sync(0xffffffffu, upto > begin)) - 1;
        cur.row = l;
        at = __shfl_sync(0xffffffffu, upto - mine, l);
    } else {
        long long mine = 0;
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
        if (blockIdx.x == 0) {
            long long x = before - mine;
            for (int i = threadIdx.x * run; i < min(a.rows, (int)(threadIdx.x + 1) * run); i++) {
                a.prefix[i] = x;
                x += row_records(i);
            }
            if (threadIdx.x == 0) a.prefix[a.rows] = s.sums[kSplitThreads];
        }
        records = s.sums[kSplitThreads];
        const Shares shares(records);
        if (worker >= shares.workers) return;
        const long long begin = shares.start(worker);
        int lo = 0, hi = kSplitThreads;  // the run: sums[lo] <= begin < sums[hi]
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
    const Shares shares(records);
    const long long begin = shares.start(worker), end = shares.start(worker + 1);

    // the first record's item and page
    row_pages(a, cur.row, cur.first, cur.last);
    long long item_at;  // record index of the current item's first page
    {
        const int pages = cur.last - cur.first;
        cur.item = (int)quotient(begin - at, pages);
        item_at = at + (long long)cur.item * pages;
        cur.page = cur.first + (int)(begin - item_at);
    }
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

    SplitQuery<kWide, kSplit> q;
    SplitState<kWide> st;
    load_query<T, kWide, kSplit>(a, cur.row, cur.item, lane, q);
    st.clear();
    int len = a.row_len[cur.row];
    int piece = 0;           // this worker's pieces: 0 starts at its first record, 1 is a later one
    uint32_t phases = 0;     // parity of each stage's next completed copy
    bool timed_out = false;
    int stage = 0;
    for (long long rec = begin; rec < end; rec++) {
        if (bad >> stage & 1) {
#pragma unroll
            for (int r = 0; r < R; r++) st.total[r] = __int_as_float(0x7fc00000);
            if (lane == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        } else {
            const bool ok = mbar_wait_bounded(&s.full[warp][stage], phases >> stage & 1, kSplitWait);
            if (!__all_sync(0xffffffffu, ok)) {
                timed_out = true;
                break;
            }
            phases ^= 1u << stage;
            const int at = cur.page * kPagePositions;
            attend_page<kWide, kSplit>(s.ring[warp][stage], a.window ? len - a.window - at : 0, len - at, lane, q, st);
        }
        __syncwarp();
        if (next < end) issue(stage);
        stage = stage + 1 == kSplitStages ? 0 : stage + 1;

        const bool item_ends = cur.page + 1 == cur.last;
        if (item_ends || rec + 1 == end) {
            // the item, or this worker's piece of it
            const bool alone = item_ends && item_at >= begin;
            const int kv = cur.item / a.blocks, block = cur.item - kv * a.blocks;
            const float back = pow2(st.exponent - 8);
#pragma unroll
            for (int r = 0; r < R; r++) {
                float total = st.total[r];
                total += __shfl_xor_sync(0xffffffffu, total, 1);
                total += __shfl_xor_sync(0xffffffffu, total, 2);
                const float inverse = 1.0f / total;
                const int in_block = r * 8 + (lane >> 2), in_group = block * kHeadBlock + in_block;
                if (in_group >= a.group) continue;
                if (alone) {
                    T *dst = static_cast<T *>(a.out) + (size_t)cur.row * a.out_stride +
                             ((size_t)kv * a.group + in_group) * kHeadDim + 2 * (lane & 3);
#pragma unroll
                    for (int D = 0; D < 8; D++)
                        store2(dst + 8 * D, st.o[D][2 * r] * inverse * back, st.o[D][2 * r + 1] * inverse * back);
                } else {
                    float *dst = a.pieces + (((size_t)worker * 2 + piece) * a.piece_heads + in_block) * kPieceHead;
#pragma unroll
                    for (int D = 0; D < 8; D++)
                        *reinterpret_cast<float2 *>(dst + 8 * D + 2 * (lane & 3)) =
                            make_float2(st.o[D][2 * r] * inverse * back, st.o[D][2 * r + 1] * inverse * back);
                    if ((lane & 3) == 0)
                        *reinterpret_cast<float2 *>(dst + kHeadDim) = make_float2(st.top[r] * q.factor[r], total);
                }
            }
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
                load_query<T, kWide, kSplit>(a, cur.row, cur.item, lane, q);
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
}

// Joins the pieces of an item in worker order,
//   out = sum w_i o_i / sum w_i,  w_i = l_i 2^(m_i - max m),
// and writes the rows that have no records.  A CTA takes an item's heads, or
// with `split_heads` one of them; its warps share out the heads, and what is
// left of them the pieces of a head, whose loads go out in batches.
template <class T>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(SplitArgs a, int split_heads) {
    constexpr int kWarps = kJoinThreads / 32, kBatch = 8;
    __shared__ float acc[kWarps][kHeadDim];
    __shared__ float2 part_ml[kWarps];
    pdl_wait();
    const int virtual_heads = a.c.heads * a.blocks;
    const int unit = split_heads ? blockIdx.x / a.piece_heads : blockIdx.x;
    const int row = unit / virtual_heads, item = unit - row * virtual_heads;
    const int kv = item / a.blocks, block = item - kv * a.blocks;
    const int first_head = split_heads ? blockIdx.x - unit * a.piece_heads : 0;
    const int heads = min(split_heads ? 1 : kHeadBlock, a.group - block * kHeadBlock - first_head);
    if (heads <= 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T *out = static_cast<T *>(a.out) + (size_t)row * a.out_stride +
             ((size_t)kv * a.group + block * kHeadBlock + first_head) * kHeadDim;
    const long long before = a.prefix[row], records = a.prefix[a.rows];
    const long long pages = quotient(a.prefix[row + 1] - before, virtual_heads);
    if (pages == 0) {
        int first, last;
        const bool good = row_pages(a, row, first, last);
        if (!good && threadIdx.x == 0 && a.c.status) atomicOr(a.c.status, kStatusBadPage);
        for (int i = threadIdx.x; i < heads * kHeadDim; i += kJoinThreads)
            out[i] = from_float<T>(good ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    const Shares shares(records);
    const long long begin = before + item * pages, end = begin + pages;
    // the workers whose ranges hold its first and last record
    const int w0 = shares.holder(begin), w1 = shares.holder(end - 1);
    if (w0 == w1) return;  // that worker wrote it
    const int first_piece = shares.start(w0) == begin ? 0 : 1;
    const int parts = heads >= kWarps ? 1 : kWarps / heads;       // warps a head
    const int count = w1 - w0 + 1, per = (count + parts - 1) / parts;
    const int part = warp % parts, from = w0 + part * per, to = min(w1 + 1, from + per);
    for (int h0 = 0; h0 < heads; h0 += kWarps / parts) {
        const int h = h0 + warp / parts;
        float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        if (h < heads) {
            const auto piece = [&](int w) {
                return a.pieces + (((size_t)w * 2 + (w == w0 ? first_piece : 0)) * a.piece_heads + first_head + h) * kPieceHead;
            };
            for (int base = from; base < to; base += kBatch) {
                float2 ml[kBatch], v[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    const bool there = base + j < to;
                    const float *p = piece(there ? base + j : from);
                    ml[j] = there ? *reinterpret_cast<const float2 *>(p + kHeadDim) : make_float2(-INFINITY, 0.0f);
                    v[j] = *reinterpret_cast<const float2 *>(p + 2 * lane);
                }
                float m = top;
#pragma unroll
                for (int j = 0; j < kBatch; j++) m = fmaxf(m, ml[j].x);
                const float keep = top == m ? 1.0f : exp2f(top - m);
                sum *= keep, o0 *= keep, o1 *= keep;
                top = m;
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    if (base + j >= to) break;
                    const float f = ml[j].x == m ? ml[j].y : ml[j].y * exp2f(ml[j].x - m);
                    sum += f, o0 = fmaf(f, v[j].x, o0), o1 = fmaf(f, v[j].y, o1);
                }
            }
        }
        if (parts > 1) {  // the warps of a head, in order (heads < kWarps: one round)
            acc[warp][2 * lane] = o0, acc[warp][2 * lane + 1] = o1;
            if (lane == 0) part_ml[warp] = make_float2(top, sum);
            __syncthreads();
            if (part != 0 || h >= heads) return;
            float m = -INFINITY;
            for (int i = 0; i < parts; i++) m = fmaxf(m, part_ml[warp + i].x);
            sum = o0 = o1 = 0.0f;
            for (int i = 0; i < parts; i++) {
                const float2 ml = part_ml[warp + i];
                if (w0 + i * per > w1) continue;  // no pieces
                const float f = ml.x == m ? 1.0f : exp2f(ml.x - m);
                sum += ml.y * f, o0 += acc[warp + i][2 * lane] * f, o1 += acc[warp + i][2 * lane + 1] * f;
            }
        }
        if (h < heads) store2(out + h * kHeadDim + 2 * lane, o0 / sum, o1 / sum);
    }
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

static size_t prefix_bytes(int rows) { return (((size_t)rows + 1) * sizeof(long long) + 15) & ~size_t(15); }

}  // namespace ndl

using namespace ndl;

// The records before each row, and two pieces a worker.
extern "C" NDL_API size_t ndl_attention_split_workspace(int rows, int heads, int kv_heads, int max_pages) {
    if (rows <= 0 || heads <= 0 || kv_heads <= 0 || max_pages <= 0 || heads % kv_heads != 0) return 0;
    const int held = heads / kv_heads < kHeadBlock ? heads / kv_heads : kHeadBlock;
    return prefix_bytes(rows) + (size_t)kSplitWorkers * 2 * held * kPieceHead * sizeof(float);
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
    SplitArgs a{q, out, q_stride, out_stride, row_slot, row_len, rows, heads, group,
                (group + kHeadBlock - 1) / kHeadBlock, window, group < kHeadBlock ? group : kHeadBlock, scale,
                {page_table, const_cast<uint8_t *>(pool), (long long)page_bytes, slots, max_pages, num_pages, layer,
                 kv_heads, status},
                static_cast<long long *>(workspace),
                reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + prefix_bytes(rows))};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const auto kernel = group > 8 ? attention_split_kernel<T, true> : attention_split_kernel<T, false>;
        constexpr size_t smem = sizeof(SplitSmem) + 128;
        static DeviceOnce attribute;  // the attributes belong to the kernels on one device
        const int st = attribute.run([&] {
            for (const auto k : {attention_split_kernel<T, true>, attention_split_kernel<T, false>}) {
                const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
                if (e != cudaSuccess)
                    return set_error(NDL_ERR_CUDA, "split attention smem: %s", cudaGetErrorString(e));
            }
            return (int)NDL_OK;
        });
        if (st != NDL_OK) return st;
        kernel<<<kSplitCtas, kSplitThreads, smem, (cudaStream_t)stream>>>(a);
        const int rc2 = check_launch("attention_split");
        if (rc2 != NDL_OK) return rc2;
        PdlScope early(true);  // the join's launch overlaps the kernel above; it waits for its end before reading
        // few items may have many pieces each: a CTA a head then
        const long long items = (long long)rows * kv_heads * a.blocks;
        const int split_heads = items < kJoinItems;
        launch_kernel(attention_join_kernel<T>, dim3((unsigned)(items * (split_heads ? a.piece_heads : 1))),
                      dim3(kJoinThreads), 0, (cudaStream_t)stream, a, split_heads);
        return check_launch("attention_join");
    });
}
