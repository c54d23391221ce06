// Log-sum-exp merge of an output row's split partials by warps.
//
// A warp takes 128 (at head_dim 64: 64) columns of a row and walks its partials 32 at a time: every lane forms the weight
// of one of them, and the columns are summed with the weights handed round by shuffles, so that a partial costs a lane one
// load and four FMAs. (With every thread forming every weight a merge of 1024 rows of 21 partials was bound by instructions:
// 12.7 us against 9.) `groups` sets of warps, a power of two, share a row where there are few rows, and join at the end.
#pragma once

#include "tt_sm100.h"

namespace {

template <int HD>
struct RowMerge {
    static constexpr int kVec = HD >= 128 ? 4 : 2;
    static constexpr uint32_t kRowWarps = HD / (32 * kVec), kSets = 8 / kRowWarps;     // of a CTA of 8 warps
    struct Columns { float v[kVec]; };
    struct Shared {
        Columns acc[256];
        float m[8], d[8];
    };

    uint32_t warp, lane, groups, grp, col;
    float m_run, d_run;
    Columns acc;

    // the row that a warp of merge CTA `block` works on
    static __device__ __forceinline__ uint32_t row(uint32_t block, uint32_t warp, uint32_t groups) {
        return block * (kSets / groups) + warp / kRowWarps / groups;
    }
    __device__ __forceinline__ RowMerge(uint32_t w, uint32_t l, uint32_t g)
        : warp(w), lane(l), groups(g), grp((w / kRowWarps) & (g - 1)), col((w % kRowWarps * 32 + l) * kVec), m_run(-INFINITY), d_run(0.f) {
#pragma unroll
        for (int x = 0; x < kVec; ++x) acc.v[x] = 0.f;
    }
    static __device__ __forceinline__ Columns load(const float *p) {
        Columns c;
        if constexpr (kVec == 4) {
            const float4 x = *reinterpret_cast<const float4 *>(p);
            c.v[0] = x.x; c.v[1] = x.y; c.v[2] = x.z; c.v[3] = x.w;
        } else {
            const float2 x = *reinterpret_cast<const float2 *>(p);
            c.v[0] = x.x; c.v[1] = x.y;
        }
        return c;
    }
    // partials base, base + stride, ... (n of them; m in natural-log domain): this set's share of them
    __device__ __forceinline__ void walk(const float *po, const float *pm, const float *pl, size_t base, size_t stride, uint32_t n) {
        for (uint32_t c0 = grp; c0 < n; c0 += 32 * groups) {
            const uint32_t count = min(32u, (n - c0 + groups - 1) / groups);
            const size_t row0 = base + (size_t)c0 * stride, step = stride * groups;
            float e = -INFINITY, l = 0.f;
            if (lane < count) { e = pm[row0 + lane * step]; l = pl[row0 + lane * step]; }
            float mx = e;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m_run, mx);
            if (m_new == -INFINITY) continue;                          // nothing visible so far: exp(-inf - -inf) would be NaN
            const float sc = __expf(m_run - m_new), wgt = __expf(e - m_new);
            float d = l * wgt;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
            d_run = d_run * sc + d;
            m_run = m_new;
#pragma unroll
            for (int x = 0; x < kVec; ++x) acc.v[x] *= sc;
            const float *p = po + row0 * HD + col;
#pragma unroll 8
            for (uint32_t i = 0; i < count; ++i, p += step * HD) {
                const float wi = __shfl_sync(0xffffffffu, wgt, i);
                const Columns o = load(p);
#pragma unroll
                for (int x = 0; x < kVec; ++x) acc.v[x] = fmaf(o.v[x], wi, acc.v[x]);
            }
        }
    }
    // Joins the sets of a row (all threads of the CTA call it); false for those whose part is done.
    __device__ __forceinline__ bool join(Shared &sh) {
        if (groups == 1) return true;
        sh.acc[warp * 32 + lane] = acc;
        if (lane == 0) { sh.m[warp] = m_run; sh.d[warp] = d_run; }
        __syncthreads();
        if (grp != 0) return false;
        float mg = m_run;
        for (uint32_t g = 1; g < groups; ++g) mg = fmaxf(mg, sh.m[warp + g * kRowWarps]);
        if (mg != -INFINITY) {
            const float sc = __expf(m_run - mg);
            d_run *= sc;
#pragma unroll
            for (int x = 0; x < kVec; ++x) acc.v[x] *= sc;
            for (uint32_t g = 1; g < groups; ++g) {
                const float wgt = __expf(sh.m[warp + g * kRowWarps] - mg);
                const Columns o = sh.acc[(warp + g * kRowWarps) * 32 + lane];
#pragma unroll
                for (int x = 0; x < kVec; ++x) acc.v[x] = fmaf(o.v[x], wgt, acc.v[x]);
                d_run += sh.d[warp + g * kRowWarps] * wgt;
            }
        }
        return true;
    }
    template <typename T>
    __device__ __forceinline__ void store(T *row_out) const {
        const float inv = d_run > 0.f ? 1.f / d_run : 0.f;             // a row that sees nothing: zeros
#pragma unroll
        for (int x = 0; x < kVec; x += 2) *reinterpret_cast<uint32_t *>(row_out + col + x) = pack2<T>(acc.v[x] * inv, acc.v[x + 1] * inv);
    }
};

// Sets of warps per row -- as many as keep two CTAs an SM busy, or four where each still has eight of a row's `parts`
// partials (1024 rows of 18 to 26: a call of 61.3 us became one of 58.3; 512 rows of nine: 208.6 and 210) -- and the CTAs that
// take `rows` rows.
inline uint32_t merge_groups(uint32_t rows, uint32_t parts, uint32_t head_dim, uint32_t sm_count, uint32_t *ctas) {
    const uint32_t sets = head_dim == 256 ? 4 : 8;
    uint32_t groups = 1;
    while (groups < sets && (uint64_t)rows * groups * 2 <= (uint64_t)sets * (parts >= 16 * groups ? 4 : 2) * sm_count) groups *= 2;
    *ctas = (uint32_t)(((uint64_t)rows * groups + sets - 1) / sets);
    return groups;
}

}  // namespace
