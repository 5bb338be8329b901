// Attention of one (row, head) over a slot's pages by one warp, fp32 throughout.
#pragma once
#include "paged.cuh"

namespace ndl {

// lanes hold dims lane and lane + 32 of q (scaled) and of the result
__device__ __forceinline__ bool attend_row(const PagedCache &c, int slot, int head, int first, int last, float *q,
                                           float &o0, float &o1, int lane) {
    float m = -INFINITY, l = 0.0f;
    o0 = o1 = 0.0f;
    bool ok = true;
    for (int base = first & ~63; base < last; base += 64) {
        const int page = cache_page(c, slot, base >> 6);
        if (page < 0) {
            ok = false;
            break;
        }
        const uint8_t *rec = cache_record(c, page, head);
        float s[2];
        for (int h = 0; h < 2; h++) {
            const int p = lane + 32 * h;
            float d = 0.0f;
            for (int i = 0; i < 64; i++) d += q[i] * (float)(int8_t)rec[k_byte(p, i)];
            s[h] = base + p >= first && base + p < last
                       ? d * reinterpret_cast<const float *>(rec + kKScaleOffset)[k_scale_index(p)]
                       : -INFINITY;
        }
        float mx = fmaxf(s[0], s[1]);
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
        const float mn = fmaxf(m, mx);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float corr = expf(m - ref);
        m = mn;
        float e[2] = {base + lane >= first && base + lane < last ? expf(s[0] - ref) : 0.0f,
                      base + lane + 32 >= first && base + lane + 32 < last ? expf(s[1] - ref) : 0.0f};
        l = l * corr + e[0] + e[1];
        o0 *= corr, o1 *= corr;
        for (int p = 0; p < 64; p++) {
            const float w = __shfl_sync(~0u, e[p >> 5], p & 31);
            if (base + p < first || base + p >= last) continue;
            const float ws = w * reinterpret_cast<const float *>(rec + kVScaleOffset)[v_scale_index(p)];
            o0 += ws * (float)(int8_t)rec[v_byte(p, lane)];
            o1 += ws * (float)(int8_t)rec[v_byte(p, lane + 32)];
        }
    }
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
    if (last > first) o0 /= l, o1 /= l;
    return ok;
}

}  // namespace ndl
