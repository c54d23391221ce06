// Decode attention of sessions that share a long prefix.
//
// The sessions of a group continue the same tokens (a system prompt, a document, the branches of one search), so the
// prefix's K/V rows exist once and every session's query rows see all of them. A batched decode would stream them once
// per session; here the query rows of the whole group are packed into one operand and the prefix is streamed once per
// 128 of them:
//
//   prefix pass   attn_prefix_kernel: (group, kv head, 128 packed rows, key range) per CTA on tcgen05 -> (m, l, o) partials
//   suffix pass   the split-KV decode kernel over every session's own rows                            -> (m, l, o) partials
//   merge         attn_prefix_merge_kernel: log-sum-exp over both kinds of partials of an output row
//
// The prefix pass packs row = (query row of the group) * G + g with G query heads per KV head, session after session;
// a packed row is a TMEM lane and one softmax thread, so nothing of the softmax crosses threads:
//
//   S[j%2] = Q . K_j^T   SS MMA M128 N128 K16 x HD/16     TMEM columns 0..255 (two tiles of 128 keys)
//   P_j    = exp2(S - m) tcgen05.ld -> registers -> tcgen05.st over the first half of the score tile's columns
//   O     += P_j . V_j   TS MMA M128 N128 (N64 at head_dim 64) K16 x8, per 128 head dims     TMEM columns 256..
//
// Shared memory holds Q and one ring of 16 KB slots that K and V chunks ([128 keys][64 head dims]) travel through in
// the order the products consume them: K(0) K(1) V(0) K(2) V(1) ... so that the product of tile j+1 is issued before
// the softmax of tile j is done. Every row of an item sees every key of its range: only the last tile of a prefix is
// masked. What bounds the pass depends on the rows: with up to about 256 packed rows per KV head the bytes of the
// prefix, beyond that the tensor pipe and the exponentials.
//
// The row maximum a tile is scaled by is only raised when a score exceeds it by more than 2^8; O is then rescaled in
// TMEM once P.V of the tile before has retired. Row sums are taken over the ROUNDED weights P.V uses, so O / l is a
// convex combination of V rows. Every mbarrier wait is bounded.
#include "tt_sm100.h"

#include <type_traits>

namespace {

constexpr int kBK = 128;                       // keys per tile
constexpr int kSlotBytes = kBK * 64 * 2;       // [128 keys][64 head dims], 128-byte rows
constexpr int kMaxSlots = 12;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRaiseThreshold = 8.0f;
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;
constexpr uint32_t kParamGroups = 8;

// Query rows of one session, in call order.
struct PrefixSession {
    const void *q;
    uint32_t first_row;     // query rows of the call before this session
    uint32_t q_rows;
};
// One group. Its items are [part][kv head][row tile].
struct PrefixGroup {
    uint32_t prefix_len, n_parts, part_len;
    uint32_t session_begin, session_count;
    uint32_t row_begin, n_rows;          // query rows of the call before the group, and its own
    uint32_t partial_base;               // first partial row
    uint32_t item_begin;
    uint32_t row_tiles;
};
struct alignas(64) PrefixMaps { unsigned char m[2][128]; };    // K and V tensor maps of a group

// Calls of up to kParamGroups groups and kParamSessions sessions carry their tables and tensor maps in the kernel
// parameters; larger ones read the copies the host uploaded.
struct alignas(64) PrefixTable {
    PrefixMaps maps[kParamGroups];
    PrefixGroup g[kParamGroups];
    PrefixSession s[kParamSessions];
    uint32_t n_groups, n_sessions;
    uint32_t in_params;
};

struct PrefixParams {
    const PrefixGroup *groups;           // device copies, when !in_params
    const PrefixSession *sessions;
    const PrefixMaps *maps;
    float *part_o, *part_m, *part_l;
    uint32_t n_q_heads, n_kv_heads, q_row_stride;
    float scale_log2;
    uint32_t idesc_qk, idesc_pv;
};

// Geometry for ROWS packed rows (64 or 128): one softmax warp per 32 rows, the producer warp, the MMA warp.
template <int HD, int ROWS>
struct PrefixGeom {
    static constexpr int kSoftmaxWarps = ROWS / 32;
    static constexpr int kProducerWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1;
    static constexpr int kThreads = (kSoftmaxWarps + 2) * 32;
    static constexpr int kChunks = HD / 64;                     // ring units of one K or V tile
    static constexpr int kQSub = ROWS * 64 * 2;
    // the M = 128 products read rows ROWS..127 of the Q operand from what follows it in shared memory (their lanes are
    // never read), so the ring must follow Q directly
    static constexpr int kSlots = ROWS == 64 || HD < 256 ? 12 : 10;
    static constexpr int kOffRing = kQSub * kChunks;
    static constexpr int kOffMisc = kOffRing + kSlots * kSlotBytes;
};

struct Misc {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t s_full[2];
    uint64_t p_ready[2];        // one arrive per softmax warp
    uint64_t o_ready[2];        // [tile parity]: the softmax threads may be two P.V products ahead of the tensor pipe when
                                // they reach the epilogue, and one barrier's parity cannot tell tile n-1 from tile n-3
    const void *row_q[128];     // where each packed row's query starts (null: no such row)
    uint32_t tmem_base;
    uint32_t pad;
};
template <int HD, int ROWS>
constexpr int prefix_smem_bytes() { return PrefixGeom<HD, ROWS>::kOffMisc + (int)sizeof(Misc) + 1024 /*align*/; }
static_assert(prefix_smem_bytes<256, 64>() <= 232448 && prefix_smem_bytes<256, 128>() <= 232448 && prefix_smem_bytes<128, 128>() <= 232448,
              "the prefix kernel's shared memory exceeds the per-CTA limit");

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(PrefixGeom<HD, ROWS>::kThreads, 1)
attn_prefix_kernel(PrefixParams p, uint32_t *__restrict__ status, const __grid_constant__ PrefixTable table) {
    using G = PrefixGeom<HD, ROWS>;
    constexpr int kSlots = G::kSlots, kThreads = G::kThreads, kQSub = G::kQSub, kChunks = G::kChunks;
    extern __shared__ unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char *q_s = smem;
    unsigned char *ring = smem + G::kOffRing;
    Misc *ms = reinterpret_cast<Misc *>(smem + G::kOffMisc);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- the item: (group, part, kv head, row tile) from the block index ----
    pdl_launch_dependents();
    pdl_wait();       // the kernel before this one may have produced the query rows
    const PrefixGroup *groups = table.in_params ? table.g : p.groups;
    const PrefixSession *sessions = table.in_params ? table.s : p.sessions;
    uint32_t gi = 0;
    {
        uint32_t hi = table.n_groups;
        while (hi - gi > 1) {
            const uint32_t mid = (gi + hi) >> 1;
            if (groups[mid].item_begin <= blockIdx.x) gi = mid; else hi = mid;
        }
    }
    const PrefixGroup grp = groups[gi];
    const uint32_t local = blockIdx.x - grp.item_begin;
    const uint32_t row_tile = local % grp.row_tiles, kv_head = local / grp.row_tiles % p.n_kv_heads;
    const uint32_t part = local / (grp.row_tiles * p.n_kv_heads);
    const uint32_t key_begin = min(grp.prefix_len, part * grp.part_len);
    const uint32_t key_end = min(grp.prefix_len, key_begin + grp.part_len);
    const uint32_t n_tiles = (key_end - key_begin + kBK - 1) / kBK;
    const uint32_t group = p.n_q_heads / p.n_kv_heads;
    const uint32_t row0 = row_tile * ROWS;                                  // first packed row of the tile
    const uint32_t n_rows = min((uint32_t)ROWS, grp.n_rows * group - row0);

    // Ring unit u (16 KB) in consumption order: K(0) | K(1) V(0) | K(2) V(1) | ... | V(n-1), kChunks units each.
    const CUtensorMap *k_map = reinterpret_cast<const CUtensorMap *>(table.in_params ? table.maps[gi].m[0] : p.maps[gi].m[0]);
    const CUtensorMap *v_map = reinterpret_cast<const CUtensorMap *>(table.in_params ? table.maps[gi].m[1] : p.maps[gi].m[1]);
    const uint32_t n_units = 2 * kChunks * n_tiles;
    auto load_unit = [&](uint32_t u) {
        const uint32_t blk = u / kChunks, c = u % kChunks;
        bool is_k; uint32_t tile;
        if (blk == 0) { is_k = true; tile = 0; }
        else if (blk == 2 * n_tiles - 1) { is_k = false; tile = n_tiles - 1; }
        else if (blk & 1) { is_k = true; tile = (blk + 1) >> 1; }
        else { is_k = false; tile = (blk >> 1) - 1; }
        const uint32_t slot = u % kSlots;
        mbar_expect_tx(&ms->full[slot], kSlotBytes);
        tma_load_2d(ring + slot * kSlotBytes, is_k ? k_map : v_map, (int)(kv_head * HD + c * 64), (int)(key_begin + tile * kBK),
                    &ms->full[slot]);
    };
    // The first ring fill leaves before anything else, so that it overlaps the arrival of Q.
    if (threadIdx.x == G::kProducerWarp * 32) {
        for (int s = 0; s < kSlots; ++s) { mbar_init(&ms->full[s], 1); mbar_init(&ms->empty[s], 1); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&ms->s_full[s], 1);
            mbar_init(&ms->p_ready[s], G::kSoftmaxWarps);
            mbar_init(&ms->o_ready[s], 1);
        }
        mbar_fence_init();
        if (!table.in_params) {
            // the maps were rewritten by a host copy since the last launch that used these addresses
            asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(k_map) : "memory");
            asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(v_map) : "memory");
        }
        for (uint32_t u = 0; u < (uint32_t)kSlots && u < n_units; ++u) load_unit(u);
    }
    // where the tile's rows come from: a search over the group's sessions, one thread per row
    for (uint32_t r = threadIdx.x; r < (uint32_t)ROWS; r += kThreads) {
        const void *src = nullptr;
        if (r < n_rows) {
            const uint32_t packed = row0 + r, qrow = grp.row_begin + packed / group;
            uint32_t lo = grp.session_begin, hi = grp.session_begin + grp.session_count;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (sessions[mid].first_row <= qrow) lo = mid; else hi = mid;
            }
            src = reinterpret_cast<const T *>(sessions[lo].q) + (size_t)(qrow - sessions[lo].first_row) * p.q_row_stride +
                  (size_t)(kv_head * group + packed % group) * HD;
        }
        ms->row_q[r] = src;
    }
    if (warp == G::kProducerWarp) {
        __syncwarp();
        tmem_alloc(&ms->tmem_base, kTmemCols);
    }
    __syncthreads();
    // ---- Q: K-major, 128-byte swizzle, 64-wide sub-tiles ----
    for (uint32_t c = threadIdx.x; c < ROWS * (HD / 8); c += kThreads) {
        const uint32_t r = c / (HD / 8), chunk = c % (HD / 8);              // 16-byte chunk of the row
        unsigned char *dst = q_s + (chunk >> 3) * kQSub + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
        const T *src = reinterpret_cast<const T *>(ms->row_q[r]);
        if (src != nullptr)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src + chunk * 8) : "memory");
        else
            *reinterpret_cast<uint4 *>(dst) = make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ms->tmem_base;
    bool failed = false;

    if (warp == G::kProducerWarp) {
        // ------------------------------------------------------------------ TMA producer
        if (lane == 0) {
            bool ok = true;
            uint32_t u = kSlots;
            for (; ok && u < n_units; ++u) {
                ok = mbar_wait(&ms->empty[u % kSlots], ((u / kSlots) - 1) & 1);
                if (ok) load_unit(u);
            }
            if (!ok) {
                // give the copies still in flight a bounded chance to land before the shared memory is released
                --u;
                for (uint32_t v = u > (uint32_t)kSlots ? u - kSlots : 0; v < u; ++v)
                    mbar_wait(&ms->full[v % kSlots], (v / kSlots) & 1, 1u << 16);
            }
            failed = !ok;
        }
    } else if (warp == G::kMmaWarp) {
        // ------------------------------------------------------------------ MMA issuer
        if (lane == 0 && n_tiles > 0) {
            const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(q_s);
            uint32_t u = 0;
            auto issue_qk = [&](uint32_t j) {
                const uint32_t d = tmem + kColS + (j & 1) * kBK;
                for (uint32_t c = 0; c < (uint32_t)kChunks; ++c, ++u) {
                    const uint32_t slot = u % kSlots;
                    if (!mbar_wait(&ms->full[slot], (u / kSlots) & 1)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint64_t ad = make_desc(q_a + c * kQSub + ks * 32, 16, 1024);
                        const uint64_t bd = make_desc(ring_a + slot * kSlotBytes + ks * 32, 16, 1024);
                        mma_ss(d, ad, bd, p.idesc_qk, (c > 0 || ks > 0) ? 1u : 0u);
                    }
                    mma_commit(&ms->empty[slot]);
                }
                mma_commit(&ms->s_full[j & 1]);
                return true;
            };
            bool ok = issue_qk(0);
            for (uint32_t j = 0; ok && j < n_tiles; ++j) {
                if (j + 1 < n_tiles) ok = issue_qk(j + 1);
                if (ok) ok = mbar_wait(&ms->p_ready[j & 1], (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t p_t = tmem + kColS + (j & 1) * kBK;    // P_j: 64 columns of 16-bit pairs over S_j
                // O(128 head dims) += P_j . V_j: V as the MN-major B operand, 64-wide head-dim atoms one slot apart
                // (LBO), 8-key groups 1024 B apart (SBO), 16 keys (2048 B) per step
                constexpr uint32_t kUnits = kChunks == 1 ? 1 : 2;      // ring units per product
                for (uint32_t c = 0; ok && c < (uint32_t)kChunks; c += kUnits, u += kUnits) {
                    const uint32_t slot = u % kSlots;
                    for (uint32_t x = 0; ok && x < kUnits; ++x) ok = mbar_wait(&ms->full[slot + x], (u / kSlots) & 1);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk) {
                        const uint64_t bd = make_desc(ring_a + slot * kSlotBytes + kk * 2048, kSlotBytes, 1024);
                        mma_ts(tmem + kColO + c * 64, p_t + kk * 8, bd, p.idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                    }
                    for (uint32_t x = 0; x < kUnits; ++x) mma_commit(&ms->empty[slot + x]);
                }
                if (!ok) break;
                mma_commit(&ms->o_ready[j & 1]);
            }
            failed = !ok;
        }
    } else {
        // ------------------------------------------------------------------ softmax: one packed row per thread
        const uint32_t row = warp * 32 + lane;                   // row of the tile == TMEM lane
        const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
        const bool row_valid = row < n_rows;
        float m_ref = -INFINITY, l_run = 0.f;                    // log2-domain reference maximum, running row sum
        bool ok = true;
        for (uint32_t j = 0; j < n_tiles; ++j) {
            const uint32_t st = j & 1;
            ok = warp_all(mbar_wait(&ms->s_full[st], (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_addr = tmem + lane_addr + kColS + st * kBK;
            uint32_t raw[4][32];
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) tmem_ld32(s_addr + c4 * 32, raw[c4]);
            tmem_wait_ld();
            const uint32_t valid = key_end - (key_begin + j * kBK);          // keys of the tile, 128 or (last tile) fewer
            if (valid < (uint32_t)kBK) {
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if ((uint32_t)(c4 * 32 + c) >= valid) raw[c4][c] = 0xff800000u;
            }
            float mx4[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) mx4[x] = fmaxf(__uint_as_float(raw[0][x]), __uint_as_float(raw[1][x]));
#pragma unroll
            for (int x = 0; x < 4; ++x) mx4[x] = fmaxf(mx4[x], fmaxf(__uint_as_float(raw[2][x]), __uint_as_float(raw[3][x])));
#pragma unroll
            for (int c = 4; c < 32; ++c)
                mx4[c & 3] = fmaxf(mx4[c & 3], fmaxf(fmaxf(__uint_as_float(raw[0][c]), __uint_as_float(raw[1][c])),
                                                     fmaxf(__uint_as_float(raw[2][c]), __uint_as_float(raw[3][c]))));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
            const float m_new = fmaxf(m_ref, mx);
            // lazy rescale: keep the stale reference while it is within 2^8 of the true maximum
            const bool raise = (m_new - m_ref > kRaiseThreshold) || (m_ref == -INFINITY && m_new != -INFINITY);
            if (j == 0) {
                m_ref = m_new;
            } else if (__any_sync(0xffffffffu, raise)) {
                // O holds the sum over tiles < j; it may only be touched once P.V of tile j-1 has retired
                ok = warp_all(mbar_wait(&ms->o_ready[(j - 1) & 1], ((j - 1) >> 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const float factor = raise ? fast_exp2(m_ref - m_new) : 1.f;
                if (raise) { l_run *= factor; m_ref = m_new; }
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lane_addr + kColO + c0, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * factor);
                    tmem_st32(tmem + lane_addr + kColO + c0, o);
                }
            }
            const float neg_m = (m_ref == -INFINITY) ? 0.f : -m_ref;
            float rs4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float p0 = fast_exp2(fmaf(__uint_as_float(raw[c4][2 * c]), p.scale_log2, neg_m));
                    const float p1 = fast_exp2(fmaf(__uint_as_float(raw[c4][2 * c + 1]), p.scale_log2, neg_m));
                    pk[c] = pack2<T>(p0, p1);       // P takes V's type: A and B of one tcgen05.mma share a format
                    rs4[c & 3] += sum2<T>(pk[c]);
                }
                tmem_st16(s_addr + c4 * 16, pk);    // over columns of this score tile that have been read above
            }
            l_run += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
            tmem_wait_st();
            tc_fence_before();                      // orders P and a rescale of O before the P.V they precede
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms->p_ready[st]);
        }

        // ---- this item's rows: O, m, l ----
        if (ok && n_tiles > 0) ok = warp_all(mbar_wait(&ms->o_ready[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1));
        if (ok) {
            tc_fence_after();
            const uint32_t packed = row0 + row;
            const size_t prow = (size_t)grp.partial_base + (size_t)part * grp.n_rows * p.n_q_heads +
                                (packed / group) * p.n_q_heads + kv_head * group + packed % group;
            if (row_valid) {
                p.part_m[prow] = (n_tiles > 0 && m_ref != -INFINITY) ? m_ref * kLn2 : -INFINITY;   // natural-log domain
                p.part_l[prow] = (n_tiles > 0 && m_ref != -INFINITY) ? l_run : 0.f;
            }
            float *dst = p.part_o + prow * HD;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                if (n_tiles > 0) {
                    tmem_ld32(tmem + lane_addr + kColO + c0, o);
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = 0u;
                }
                if (row_valid) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4)
                        *reinterpret_cast<float4 *>(dst + c0 + c) =
                            make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]),
                                        __uint_as_float(o[c + 3]));
                }
            }
        }
        failed = !ok;
    }

    if (failed) atomicOr(status, TT_DEV_WAIT_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == G::kProducerWarp) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------------------------------
// Merge: one CTA per output row (session, query row, head); 256 threads are groups of HD / 4 column threads that walk
// the row's partials, the prefix's first, then the session's own, with an online (max, sum, output) triple each.
// ---------------------------------------------------------------------------------------
struct MergeSession {
    void *out;
    uint32_t first_row, q_rows;          // query rows of the call before this session, and its own
    uint32_t prefix_base, prefix_parts;  // partial rows of this session's first query row in its group's prefix pass
    uint32_t prefix_stride;              // partial rows between two parts of the prefix
    uint32_t own_base, own_parts;        // the session's own split partials
    uint32_t pad;
};
struct MergeTable {
    MergeSession s[kParamSessions];
    uint32_t n;                          // 0: the device copy
};

template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_prefix_merge_kernel(const __grid_constant__ MergeTable table, const MergeSession *__restrict__ dev, uint32_t n_sessions,
                         const float *__restrict__ pre_o, const float *__restrict__ pre_m, const float *__restrict__ pre_l,
                         const float *__restrict__ own_o, const float *__restrict__ own_m, const float *__restrict__ own_l,
                         uint32_t n_q_heads, uint32_t out_row_stride) {
    constexpr uint32_t kCols = HD / 4, kGroups = 256 / kCols;
    __shared__ float grp_m[kGroups], grp_d[kGroups];
    __shared__ float4 accs[256];
    pdl_launch_dependents();
    pdl_wait();
    const MergeSession *sessions = table.n != 0 ? table.s : dev;
    const uint32_t qrow = blockIdx.x / n_q_heads, head = blockIdx.x % n_q_heads;
    uint32_t lo = 0, hi = n_sessions;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sessions[mid].first_row <= qrow) lo = mid; else hi = mid;
    }
    const MergeSession ses = sessions[lo];
    const uint32_t w = qrow - ses.first_row;
    const uint32_t grp = threadIdx.x / kCols, ct = threadIdx.x % kCols;
    const uint32_t n_parts = ses.prefix_parts + ses.own_parts;
    const size_t pre = (size_t)ses.prefix_base + w * n_q_heads + head, own = (size_t)ses.own_base + w * n_q_heads + head;
    const size_t own_stride = (size_t)ses.q_rows * n_q_heads;

    float m_run = -INFINITY, d_run = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kBatch = 4;                             // independent loads in flight per thread
    for (uint32_t c0 = grp; c0 < n_parts; c0 += kBatch * kGroups) {
        float e[kBatch], l[kBatch]; float4 o[kBatch];
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const uint32_t c = c0 + x * kGroups;
            e[x] = -INFINITY; l[x] = 0.f; o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c < n_parts) {
                const bool shared = c < ses.prefix_parts;
                const size_t row = shared ? pre + (size_t)c * ses.prefix_stride : own + (c - ses.prefix_parts) * own_stride;
                e[x] = (shared ? pre_m : own_m)[row];
                l[x] = (shared ? pre_l : own_l)[row];
                o[x] = *reinterpret_cast<const float4 *>((shared ? pre_o : own_o) + row * HD + ct * 4);
            }
        }
        const float m_new = fmaxf(m_run, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
        if (m_new != -INFINITY) {
            const float sc = __expf(m_run - m_new);
            acc.x *= sc; acc.y *= sc; acc.z *= sc; acc.w *= sc; d_run *= sc;
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                const float wgt = __expf(e[x] - m_new);
                acc.x += o[x].x * wgt; acc.y += o[x].y * wgt; acc.z += o[x].z * wgt; acc.w += o[x].w * wgt;
                d_run += l[x] * wgt;
            }
            m_run = m_new;
        }
    }
    accs[threadIdx.x] = acc;
    if (ct == 0) { grp_m[grp] = m_run; grp_d[grp] = d_run; }
    __syncthreads();
    if (grp != 0) return;
    float mg = grp_m[0];
#pragma unroll
    for (uint32_t g = 1; g < kGroups; ++g) mg = fmaxf(mg, grp_m[g]);
    float D = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mg != -INFINITY)
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) {
            const float wgt = __expf(grp_m[g] - mg);
            const float4 o = accs[g * kCols + ct];
            acc.x += o.x * wgt; acc.y += o.y * wgt; acc.z += o.z * wgt; acc.w += o.w * wgt;
            D += grp_d[g] * wgt;
        }
    const float inv = D > 0.f ? 1.f / D : 0.f;            // a row that sees nothing: zeros
    T *dst = reinterpret_cast<T *>(ses.out) + (size_t)w * out_row_stride + (size_t)head * HD + ct * 4;
    uint2 packed;
    packed.x = pack2<T>(acc.x * inv, acc.y * inv);
    packed.y = pack2<T>(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2 *>(dst) = packed;
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// Packed rows one CTA of the prefix pass takes: 64 when no group has more, else 128.
uint32_t rows_per_tile(const uint32_t *query_rows, uint32_t n_groups, uint32_t group) {
    for (uint32_t g = 0; g < n_groups; ++g)
        if ((uint64_t)query_rows[g] * group > 64) return 128;
    return 64;
}

template <typename T, int HD, int ROWS>
cudaError_t launch_prefix_one(tt_context *ctx, cudaStream_t stream, uint32_t n_items, const PrefixParams &kp, const PrefixTable &table) {
    auto kernel = attn_prefix_kernel<T, HD, ROWS>;
    const int smem = prefix_smem_bytes<HD, ROWS>();
    cudaError_t e = tt_set_smem_once(kernel, smem);
    if (e != cudaSuccess) return e;
    return tt_launch_pdl(kernel, dim3(n_items), dim3(PrefixGeom<HD, ROWS>::kThreads), (size_t)smem, stream, kp, ctx->status, table);
}

template <typename T>
cudaError_t launch_prefix(tt_context *ctx, cudaStream_t stream, uint32_t head_dim, uint32_t rows, uint32_t n_items,
                          const PrefixParams &kp, const PrefixTable &table) {
#define TT_X(HD) (rows == 64 ? launch_prefix_one<T, HD, 64>(ctx, stream, n_items, kp, table) : launch_prefix_one<T, HD, 128>(ctx, stream, n_items, kp, table))
    return head_dim == 64 ? TT_X(64) : head_dim == 128 ? TT_X(128) : TT_X(256);
#undef TT_X
}

template <typename T>
cudaError_t launch_merge(cudaStream_t stream, uint32_t head_dim, uint32_t rows, const MergeTable &table, const MergeSession *dev,
                         uint32_t n_sessions, const PrefixParams &kp, const TTDecodeForm &own, uint32_t n_q_heads, uint32_t out_row_stride) {
#define TT_X(HD) tt_launch_pdl(attn_prefix_merge_kernel<T, HD>, dim3(rows), dim3(256), 0, stream, table, dev, n_sessions, kp.part_o, \
                               kp.part_m, kp.part_l, own.part_o, own.part_m, own.part_l, n_q_heads, out_row_stride)
    return head_dim == 64 ? TT_X(64) : head_dim == 128 ? TT_X(128) : TT_X(256);
#undef TT_X
}

}  // namespace

// The items of all groups are nearly equal slices and one CTA is resident per SM, so a launch takes about
// waves x (tiles per item + what an item costs besides its tiles), which `kItemTiles` puts at three tiles of streaming.
// The shortest such time over the part counts of the longest prefix wins; equal times go to the longer item (fewer
// partials to merge).
TT_API int tt_attn_plan_prefix_splits(const uint32_t *prefix_lens, const uint32_t *query_rows, uint32_t n_groups, uint32_t head_dim,
                                      uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t sm_count, size_t workspace_bytes,
                                      uint32_t *out_keys_per_item, uint32_t *out_n_items) {
    if (prefix_lens == nullptr || query_rows == nullptr || n_groups == 0 || n_kv_heads == 0 || n_q_heads == 0 ||
        n_q_heads % n_kv_heads != 0 || head_dim == 0 || sm_count == 0)
        return TT_ERR_INVALID_ARG;
    constexpr uint32_t kItemTiles = 3;
    const uint32_t group = n_q_heads / n_kv_heads, tile_rows = rows_per_tile(query_rows, n_groups, group);
    uint32_t longest = 0;
    for (uint32_t g = 0; g < n_groups; ++g) longest = prefix_lens[g] > longest ? prefix_lens[g] : longest;
    const uint32_t max_tiles = longest == 0 ? 1 : ceil_div(longest, kBK);
    uint64_t best = ~0ull, best_items = 0;
    uint32_t best_tiles = 0;
    for (uint32_t parts = 1; parts <= 512 && parts <= max_tiles; ++parts) {
        const uint32_t tiles = ceil_div(max_tiles, parts);
        if (parts > 1 && tiles == ceil_div(max_tiles, parts - 1)) continue;      // the same item length again
        uint64_t items = 0, prows = 0;
        for (uint32_t g = 0; g < n_groups; ++g) {
            const uint64_t p = ceil_div(prefix_lens[g], (uint64_t)tiles * kBK);
            items += p * n_kv_heads * ceil_div((uint64_t)query_rows[g] * group, tile_rows);
            prows += p * query_rows[g] * n_q_heads;
        }
        if (workspace_bytes != 0 && prows * ((uint64_t)head_dim + 2) * sizeof(float) > workspace_bytes) break;    // more parts need more
        const uint64_t time = (items + sm_count - 1) / sm_count * (tiles + kItemTiles);
        if (time < best) { best = time; best_tiles = tiles; best_items = items; }
    }
    if (best_tiles == 0) return TT_ERR_OOM;
    if (out_keys_per_item) *out_keys_per_item = best_tiles * kBK;
    if (out_n_items) *out_n_items = (uint32_t)best_items;
    return TT_OK;
}

TT_API int tt_attn_decode_shared_prefix(tt_context *ctx, tt_stream stream, const tt_attn_prefix *groups, uint32_t n_groups,
                                        const tt_attn_session *sessions, uint32_t n_sessions, const tt_attn_batch_params *params) {
    TT_ENTER(ctx);
    if (params == nullptr || ((sessions == nullptr || groups == nullptr) && n_sessions != 0))
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "groups, sessions and params must not be null");
    if (n_sessions > ctx->max_sessions)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_sessions %u exceeds the context's max_sessions %u", n_sessions, ctx->max_sessions);
    if (n_groups > ctx->max_sessions)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_groups %u exceeds the context's max_sessions %u", n_groups, ctx->max_sessions);
    if (n_sessions == 0) return TT_OK;
    const tt_attn_batch_params &q = *params;
    if (q.n_kv_heads == 0 || q.n_q_heads == 0 || q.n_q_heads % q.n_kv_heads != 0)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_q_heads must be a multiple of n_kv_heads");
    if (q.head_dim != 64 && q.head_dim != 128 && q.head_dim != 256)
        return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "decode attention supports head_dim 64/128/256, got %u", q.head_dim);
    if (!(q.scale > 0.f)) return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "a shared prefix needs a positive scale");
    if (q.kv_token_stride_elements % 8 || q.kv_token_stride_elements < q.n_kv_heads * q.head_dim)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "kv_token_stride_elements must hold a row and be a multiple of 8");
    uint64_t covered = 0;
    for (uint32_t g = 0; g < n_groups; ++g) {
        if (groups[g].n_sessions == 0) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "group %u has no sessions", g);
        if (groups[g].prefix_len > (uint32_t)INT32_MAX) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "group %u: the prefix is too long", g);
        if (groups[g].prefix_len != 0 && (groups[g].k == nullptr || groups[g].v == nullptr))
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "group %u has a null buffer", g);
        if (((uintptr_t)groups[g].k | (uintptr_t)groups[g].v) & 15)
            return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "group %u: buffers must be 16-byte aligned", g);
        covered += groups[g].n_sessions;
    }
    if (covered != n_sessions)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "the groups have %llu sessions, the call %u", (unsigned long long)covered, n_sessions);

    const bool in_params = n_groups <= kParamGroups && n_sessions <= kParamSessions;
    if (!in_params && tt_stream_is_capturing((cudaStream_t)stream))
        return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE,
                            "more than %u groups or %u sessions cannot be captured: their tables are uploaded from host memory",
                            kParamGroups, kParamSessions);
    // host tables: the parameter blocks, or the staging copy of what is uploaded
    static thread_local PrefixTable table;
    static thread_local MergeTable merge;
    const size_t off_groups = sizeof(PrefixMaps) * (size_t)n_groups, off_sessions = off_groups + sizeof(PrefixGroup) * (size_t)n_groups;
    const size_t off_merge = (off_sessions + sizeof(PrefixSession) * (size_t)n_sessions + 15) / 16 * 16;
    const size_t table_bytes = off_merge + sizeof(MergeSession) * (size_t)n_sessions;
    unsigned char *host = ctx->h_prefix_tables;
    PrefixMaps *h_maps = in_params ? table.maps : reinterpret_cast<PrefixMaps *>(host);
    PrefixGroup *h_groups = in_params ? table.g : reinterpret_cast<PrefixGroup *>(host + off_groups);
    PrefixSession *h_sessions = in_params ? table.s : reinterpret_cast<PrefixSession *>(host + off_sessions);
    MergeSession *h_merge = in_params ? merge.s : reinterpret_cast<MergeSession *>(host + off_merge);
    if (!in_params && table_bytes > ctx->prefix_table_bytes) return tt_set_error(ctx, TT_ERR_OOM, "the prefix tables do not fit the context");

    // ---- sessions, query rows per group ----
    TTDecodeSession *tmp = ctx->h_sessions_in;
    uint32_t total_rows = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        const tt_attn_session &s = sessions[i];
        if (s.kv_start != 0) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: kv_start must be 0", i);
        if (s.q == nullptr || s.out == nullptr) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u has a null buffer", i);
        if (s.q_rows == 0 || s.q_rows > 64) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: q_rows must be in 1..64", i);
        if (s.seq_len > (uint32_t)INT32_MAX || s.seq_len + 1 < s.q_rows)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: seq_len %u cannot hold %u query rows", i, s.seq_len, s.q_rows);
        if (((uintptr_t)s.q | (uintptr_t)s.out) & 15)
            return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "session %u: buffers must be 16-byte aligned", i);
        h_sessions[i].q = s.q; h_sessions[i].first_row = total_rows; h_sessions[i].q_rows = s.q_rows;
        h_merge[i].out = s.out; h_merge[i].first_row = total_rows; h_merge[i].q_rows = s.q_rows; h_merge[i].pad = 0;
        TTDecodeSession &d = tmp[i];
        d.q = s.q; d.out = s.out; d.k = s.k; d.v = s.v; d.seq_len = s.seq_len; d.q_rows = s.q_rows; d.kv_start = 0;
        d.n_parts = 0; d.partial_base = 0; d.ring_capacity = 0; d.keep = nullptr; d.row_index = nullptr;
        total_rows += s.q_rows;
    }
    uint32_t *lens = ctx->h_prefix_lens, *rows = ctx->h_prefix_rows;
    for (uint32_t g = 0, first = 0; g < n_groups; ++g) {
        lens[g] = groups[g].prefix_len;
        rows[g] = 0;
        for (uint32_t i = 0; i < groups[g].n_sessions; ++i) rows[g] += sessions[first + i].q_rows;
        first += groups[g].n_sessions;
    }
    // ---- plan: the prefix pass may take half of the workspace, at its end ----
    uint32_t keys_per_item = 0, n_items = 0;
    const size_t room = ctx->workspace_bytes / 2;
    if (tt_attn_plan_prefix_splits(lens, rows, n_groups, q.head_dim, q.n_q_heads, q.n_kv_heads, (uint32_t)ctx->sm_count, room,
                                   &keys_per_item, &n_items) != TT_OK)
        return tt_set_error(ctx, TT_ERR_OOM, "the prefix partials do not fit the context workspace");
    const uint32_t group = q.n_q_heads / q.n_kv_heads, tile_rows = rows_per_tile(rows, n_groups, group);
    uint32_t item = 0, partial = 0, session = 0, row = 0;
    for (uint32_t g = 0; g < n_groups; ++g) {
        PrefixGroup &d = h_groups[g];
        d.prefix_len = lens[g];
        d.n_parts = ceil_div(lens[g], keys_per_item);
        d.part_len = keys_per_item;
        if (d.n_parts != 0)               // parts of equal length
            d.part_len = ceil_div(ceil_div(lens[g], d.n_parts), kBK) * kBK;
        if (d.n_parts != 0) d.n_parts = ceil_div(lens[g], d.part_len);
        d.session_begin = session; d.session_count = groups[g].n_sessions;
        d.row_begin = row; d.n_rows = rows[g];
        d.partial_base = partial; d.item_begin = item;
        d.row_tiles = ceil_div((uint64_t)rows[g] * group, tile_rows);
        for (uint32_t i = 0; i < groups[g].n_sessions; ++i) {
            MergeSession &m = h_merge[session + i];
            m.prefix_base = partial + (m.first_row - row) * q.n_q_heads;
            m.prefix_parts = d.n_parts;
            m.prefix_stride = rows[g] * q.n_q_heads;
        }
        item += d.n_parts * q.n_kv_heads * d.row_tiles;
        partial += d.n_parts * rows[g] * q.n_q_heads;
        session += groups[g].n_sessions;
        row += rows[g];
        const uint64_t map_rows = lens[g] ? lens[g] : 1;
        if (lens[g] != 0 &&
            !(tt_make_tensor_map_2d(reinterpret_cast<CUtensorMap *>(h_maps[g].m[0]), groups[g].k, q.io_dtype, (uint64_t)q.n_kv_heads * q.head_dim,
                                    map_rows, q.kv_token_stride_elements, kBK) &&
              tt_make_tensor_map_2d(reinterpret_cast<CUtensorMap *>(h_maps[g].m[1]), groups[g].v, q.io_dtype, (uint64_t)q.n_kv_heads * q.head_dim,
                                    map_rows, q.kv_token_stride_elements, kBK)))
            return tt_set_error(ctx, TT_ERR_CUDA, "cuTensorMapEncodeTiled failed for group %u", g);
    }
    const size_t partial_bytes = ((size_t)partial * (q.head_dim + 2) * sizeof(float) + 255) / 256 * 256;

    // ---- suffix pass (it also checks the rest of the arguments) ----
    TTDecodeForm own;
    own.reserved_bytes = partial_bytes + 256;
    own.partials_only = true;
    int rc = tt_launch_decode(ctx, (cudaStream_t)stream, tmp, n_sessions, params, 0, nullptr, nullptr, nullptr, nullptr, nullptr, &own);
    if (rc != TT_OK) return rc;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        h_merge[i].own_base = ctx->h_sessions[i].partial_base;
        h_merge[i].own_parts = ctx->h_sessions[i].n_parts;
    }
    cudaError_t e = cudaSuccess;
    if (!in_params) {
        e = cudaMemcpyAsync(ctx->prefix_tables, host, table_bytes, cudaMemcpyHostToDevice, (cudaStream_t)stream);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "copy prefix tables");
    }
    // ---- prefix pass ----
    PrefixParams kp;
    kp.maps = reinterpret_cast<const PrefixMaps *>(ctx->prefix_tables);
    kp.groups = reinterpret_cast<const PrefixGroup *>(ctx->prefix_tables + off_groups);
    kp.sessions = reinterpret_cast<const PrefixSession *>(ctx->prefix_tables + off_sessions);
    kp.part_o = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->partials) + (ctx->workspace_bytes / 256 * 256 - partial_bytes));
    kp.part_m = kp.part_o + (size_t)partial * q.head_dim;
    kp.part_l = kp.part_m + partial;
    kp.n_q_heads = q.n_q_heads; kp.n_kv_heads = q.n_kv_heads; kp.q_row_stride = q.q_row_stride_elements;
    kp.scale_log2 = q.scale * kLog2e;
    kp.idesc_qk = tt_make_idesc_f16(q.io_dtype, kBK, false);
    kp.idesc_pv = tt_make_idesc_f16(q.io_dtype, q.head_dim == 64 ? 64 : 128, true);
    table.n_groups = n_groups; table.n_sessions = n_sessions; table.in_params = in_params ? 1u : 0u;
    merge.n = in_params ? n_sessions : 0u;
    if (item != 0) {
        e = q.io_dtype == TT_F16 ? launch_prefix<__half>(ctx, (cudaStream_t)stream, q.head_dim, tile_rows, item, kp, table)
                                 : launch_prefix<__nv_bfloat16>(ctx, (cudaStream_t)stream, q.head_dim, tile_rows, item, kp, table);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_prefix launch");
        ctx->launches++;
    }
    // ---- merge ----
    const MergeSession *dev = reinterpret_cast<const MergeSession *>(ctx->prefix_tables + off_merge);
    e = q.io_dtype == TT_F16
            ? launch_merge<__half>((cudaStream_t)stream, q.head_dim, total_rows * q.n_q_heads, merge, dev, n_sessions, kp, own, q.n_q_heads, q.out_row_stride_elements)
            : launch_merge<__nv_bfloat16>((cudaStream_t)stream, q.head_dim, total_rows * q.n_q_heads, merge, dev, n_sessions, kp, own, q.n_q_heads, q.out_row_stride_elements);
    if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_prefix_merge launch");
    ctx->launches++;
    return TT_OK;
}
