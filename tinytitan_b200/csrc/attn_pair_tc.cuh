// Attention of up to 256 query rows that share their keys, on a pair of SMs (tcgen05 cta_group::2), head_dim 256: the
// tensor-bound form of the kernel in attn_rows_tc.cuh, for shared-prefix decode with many rows (attn_prefix.cu) and for
// prefill with sinks (attn_prefill_sink.cu).
//
// One SM cannot keep its tensor pipe busy at head_dim 256: measured on this part, an M128 K16 product takes 110 clocks
// with A in shared memory and N <= 128, 66 with A in TMEM (N128) and 130 at N256 either way, so a 128-key tile is 2120
// clocks only with Q in TMEM and P.V at N256; and 128 KB of K and V per tile go into shared memory and out of it again,
// next to P, which is another 2500 clocks of its port. Two CTAs that take 128 rows each of one 256-row product need half of
// every K and V tile each: 64 KB per tile and SM, a ring that holds 2.5 tiles, and half of the L2 traffic.
//
//   S   = Q . K_j^T    TS MMA M256 N128 K16 x16   Q in TMEM columns 384..511, S in 256..383; each CTA's shared memory
//                                                 holds 64 of the tile's 128 keys
//   P_j = exp2(S - m)  TMEM -> registers -> shared memory (K-major A operand, two buffers)
//   O  += P_j . V_j    SS MMA M256 N256 K16 x8    TMEM columns 0..255; each CTA's shared memory holds 128 of the head dims
//
// Both CTAs run the same producer and softmax warps on their own rows and halves; the even CTA's two issuing threads
// (one per product) run the pair's MMAs. What they wait for arrives at the even CTA's barriers from both CTAs (TMA bytes
// through the pair's copies, softmax warps through remote arrivals), what they finish is committed to both CTAs. The
// score tile is free as soon as both CTAs hold it in registers, so Q.K^T runs up to two tiles ahead of P.V; two softmax
// groups of four warps take the tiles in turn and hand the running maximum on, as in attn_rows_tc.cuh.
//
// Measured: 2600 clocks a tile behind a prefix of 32768 keys, 2400 in a prompt's chunk whose keys are in L2 (the products
// alone 2130; TMA writes and the weights' stores share the port they are read through), 212 to 247 us over a prompt of 8192
// tokens on different machines, 0.83 to 0.71 of the sustained rate of a library product of 8192^3, and 13,000 to 15,000 clocks an item besides its tiles: 3300 to the
// cluster barrier, 1100 for Q, 3500 to 5000 to the first scores, 5500 for the output.
//
// Every mbarrier wait is bounded; all threads of both CTAs meet at the cluster barrier before TMEM is released.
#pragma once

#include "attn_rows_tc.cuh"

namespace {

constexpr int kPairThreads = 384;              // softmax groups: warps 0-3 and 4-7; 8 K producer, 9 Q.K^T issuer, 10 P.V issuer, 11 V producer
constexpr int kPairSlots = 10;                 // the first five are K's ring, the others V's
constexpr int kPairRing = kPairSlots / 2;
constexpr int kPairSlotBytes = 16384;          // two boxes [64 keys][64 head dims]
constexpr int kPairPBytes = 128 * 128 * 2;     // one buffer: two sub-tiles [128 rows][64 keys]
constexpr int kPairOffRing = 2 * kPairPBytes;  // the P buffers come first; they also take Q on its way to TMEM
constexpr int kPairOffMisc = kPairOffRing + kPairSlots * kPairSlotBytes;
constexpr int kPairStagePitch = 256 * 4 + 16;
static_assert(128 * kPairStagePitch <= kPairSlots * kPairSlotBytes, "the output tile must fit the ring");
constexpr uint32_t kPairColO = 0, kPairColS = 256, kPairColQ = 384;

struct PairShared {
    // waited for in the even CTA
    uint64_t full[kPairSlots];    // the bytes of both CTAs' halves
    uint64_t q_ready;             // one arrive per softmax warp of both CTAs: Q is in TMEM
    uint64_t s_read;              // ... of the tile's group: the scores are in registers
    uint64_t p_ready[2];          // ... of the tile's group: P is in shared memory
    // committed to both CTAs
    uint64_t empty[kPairSlots];
    uint64_t s_full[2];           // [tile parity]
    uint64_t o_ready[2];          // [tile parity]: P.V of the tile has retired, its P buffer is free
    // within a CTA
    uint64_t published[2][4];
    uint64_t pair[4];
    float l_sum[2][128];
    float m_ref[2][128];
    uint32_t tmem_base;
    uint32_t pad;
};
constexpr int kPairSmemBytes = kPairOffMisc + (int)sizeof(PairShared);
static_assert(kPairSmemBytes <= 232448, "shared memory exceeds the per-CTA limit");

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// the address of the even CTA's copy of a shared variable
__device__ __forceinline__ uint32_t even_cta_addr(const void *p) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}
__device__ __forceinline__ void mbar_arrive_even(uint64_t *bar) {
    // release at CTA scope: what the arrival publishes (TMEM, this CTA's shared memory behind a proxy fence) is read by
    // this SM's own tensor core; a cluster-scope release measured about 1000 clocks more per arrival
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(even_cta_addr(bar)) : "memory");
}
// copy into this CTA's shared memory whose bytes are counted on the even CTA's barrier
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(even_cta_addr(bar))
        : "memory");
}
__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
// completion of everything issued so far, on the barrier at this offset in both CTAs
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
}

// Bounded wait of a single thread that has nothing else to do: polls without the suspension of try_wait.
__device__ __forceinline__ bool mbar_poll(uint64_t *bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    for (uint32_t it = 0; it < 16 * kMbarWaitLimit; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(addr), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}

// The Form is that of attn_rows_kernel with ROWS = 256: rows 0..127 are the even CTA's.
template <typename T, class Form>
__global__ void __launch_bounds__(kPairThreads, 1)
attn_pair_kernel(RowsParams p, uint32_t *__restrict__ status, const __grid_constant__ Form form) {
    constexpr int HD = 256, ROWS = 256;
    extern __shared__ __align__(1024) unsigned char smem[];
    if (smem_u32(smem) & 1023u) {              // the same in both CTAs
        if (threadIdx.x == 0) atomicOr(status, TT_DEV_BAD_ITEM);
        return;
    }
    unsigned char *p_s = smem;
    unsigned char *ring = smem + kPairOffRing;
    PairShared *sh = reinterpret_cast<PairShared *>(smem + kPairOffMisc);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();

    pdl_launch_dependents();
    const typename Form::Item item = form.item(blockIdx.x >> 1, HD, ROWS);   // from the parameters alone
    if (!form.waits_late()) pdl_wait();       // the kernel before this one may have produced the query or cache rows
    const uint32_t n_tiles = item.n_tiles;                                   // >= 1
    const uint32_t my_row0 = rank * 128;

    if (threadIdx.x == 8 * 32) {
        for (int s = 0; s < kPairSlots; ++s) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        mbar_init(&sh->q_ready, 16);
        mbar_init(&sh->s_read, 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sh->p_ready[s], 8);
            mbar_init(&sh->s_full[s], 1);
            mbar_init(&sh->o_ready[s], 1);
            for (int w = 0; w < 4; ++w) mbar_init(&sh->published[s][w], 1);
        }
        for (int w = 0; w < 4; ++w) mbar_init(&sh->pair[w], 2);
        mbar_fence_init();
    }
    if (warp < 8)
        // whole rows of Q by asynchronous copies into the P buffers, 16-byte chunk c of row r at c ^ (r & 7); in flight
        // while the barriers and TMEM are set up
        load_query_rows<HD, ROWS, 16>(form, item, my_row0, warp, 8, lane, [&](uint32_t r, uint32_t chunk) {
            return p_s + r * (HD * 2) + ((chunk ^ (r & 7)) << 4);
        });
    if (warp == 8) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh->tmem_base)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();            // the barriers of both CTAs exist, and within the CTA the TMEM base is visible
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    bool failed = false;

    // Two units per tile and operand, each operand in its own ring: a slot is free as soon as its product has retired, and
    // K's slots do not wait for the softmax that V's do.
    if (warp == 8 || warp == 11) {
        // ------------------------------------------------------------------ TMA producers: this CTA's halves of K, of V
        if (lane == 0) {
            form.acquire(item);
            const bool is_k = warp == 8;
            RingPos<kPairRing> pos(0);
            const uint32_t ring0 = is_k ? 0u : kPairRing;
            // K: this CTA's 64 keys, head dims 128 half .. +127; V: keys 64 half .. +63, this CTA's 128 head dims
            const int x0 = (int)(item.kv_head * HD + (is_k ? 0 : rank * 128)), x_step = is_k ? 128 : 0;
            bool ok = true;
            uint32_t j = 0, half = 0;
            for (; j < n_tiles; ++j) {
                int row = 0;
                const CUtensorMap *map = nullptr;
                if (is_k) map = form.box(item, j, rank, true, row);
#pragma unroll 1
                for (half = 0; half < 2; ++half) {
                    if (!is_k && half == 1 && 2 * j + 1 >= item.n_halves) break;     // every key of it is hidden
                    if (!is_k) map = form.box(item, j, half, false, row);
                    const uint32_t slot = ring0 + pos.slot;
                    if (pos.lap > 0) ok = mbar_wait(&sh->empty[slot], (pos.lap - 1) & 1);
                    if (!ok) break;
                    uint64_t *bar = &sh->full[slot];
                    unsigned char *dst = ring + slot * kPairSlotBytes;
                    if (rank == 0) mbar_expect_tx(bar, 2 * kPairSlotBytes);
                    const int x = x0 + (int)half * x_step;
                    tma_load_2d_pair(dst, map, x, row, bar);
                    tma_load_2d_pair(dst + kPairSlotBytes / 2, map, x + 64, row, bar);
                    pos.advance(1);
                }
                if (!ok) break;
            }
            if (!ok && rank == 0)
                // give the copies still in flight (both CTAs') a bounded chance to land before shared memory is released
                for (uint32_t s = 0; s < (uint32_t)kPairSlots; ++s) {
                    mbar_wait(&sh->full[s], 0, 1u << 15);
                    mbar_wait(&sh->full[s], 1, 1u << 15);
                }
            failed = !ok;
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ Q.K^T issuer of the pair
        if (lane == 0 && rank == 0) {
            const uint32_t ring_a = smem_u32(ring);
            RingPos<kPairRing> pos(0);
            bool ok = mbar_wait(&sh->q_ready, 0);
            for (uint32_t j = 0; ok && j < n_tiles; ++j) {
                // the tile's K first: its wait is off the chain product -> scores read -> next product that paces the kernel
                const uint32_t slot0 = pos.slot, lap0 = pos.lap;
                pos.advance(1);
                const uint32_t slot1 = pos.slot, lap1 = pos.lap;
                pos.advance(1);
                ok = mbar_wait(&sh->full[slot0], lap0 & 1) && mbar_wait(&sh->full[slot1], lap1 & 1);
                if (ok && j > 0) ok = mbar_poll(&sh->s_read, (j - 1) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    const uint32_t slot = half ? slot1 : slot0;
                    const uint64_t bd0 = make_desc(ring_a + slot * kPairSlotBytes, 16, 1024);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        // A: 8 TMEM columns per 16-wide step; B: K-major rows of 128 bytes, 64-wide sub-tiles 8 KB apart
                        mma_ts_pair(tmem + kPairColS, tmem + kPairColQ + (half * 8 + ks) * 8, bd0 + (((ks >> 2) * 8192 + (ks & 3) * 32) >> 4),
                                    p.idesc_qk, (half > 0 || ks > 0) ? 1u : 0u);
                    mma_commit_pair(&sh->empty[slot]);
                }
                mma_commit_pair(&sh->s_full[j & 1]);
            }
            failed = !ok;
        }
    } else if (warp == 10) {
        // ------------------------------------------------------------------ P.V issuer of the pair
        if (lane == 0 && rank == 0) {
            const uint32_t ring_a = smem_u32(ring), p_a = smem_u32(p_s);
            RingPos<kPairRing> pos(0);
            bool ok = true;
            for (uint32_t j = 0; ok && j < n_tiles; ++j) {
                const uint32_t halves = 2 * j + 1 < item.n_halves ? 2 : 1;       // 1: the last tile's second half is hidden from all rows
                const uint32_t slot0 = kPairRing + pos.slot, lap0 = pos.lap;
                pos.advance(1);
                const uint32_t slot1 = kPairRing + pos.slot, lap1 = pos.lap;
                pos.advance(1);
                ok = mbar_wait(&sh->full[slot0], lap0 & 1) && (halves == 1 || mbar_wait(&sh->full[slot1], lap1 & 1));
                if (ok) ok = mbar_poll(&sh->p_ready[j & 1], (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    if (half == halves) break;
                    const uint32_t slot = half ? slot1 : slot0;
                    // P: K-major, sub-tile `half` = keys 64 half .., 16 keys (32 B) per step. V: MN-major, 64-wide
                    // head-dim atoms 8 KB apart (LBO), 8-key groups 1024 B apart (SBO), 16 keys (2048 B) per step
                    const uint64_t ad0 = make_desc(p_a + (j & 1) * kPairPBytes + half * 16384, 16, 1024);
                    const uint64_t bd0 = make_desc(ring_a + slot * kPairSlotBytes, 8192, 1024);
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4)
                        mma_ss_pair(tmem + kPairColO, ad0 + (k4 * 32 >> 4), bd0 + (k4 * 2048 >> 4), p.idesc_pv,
                                    (j > 0 || half > 0 || k4 > 0) ? 1u : 0u);
                    mma_commit_pair(&sh->empty[slot]);
                }
                mma_commit_pair(&sh->o_ready[j & 1]);
            }
            failed = !ok;
        }
    } else {
        // ------------------------------------------------------------------ Q into TMEM, then softmax
        const uint32_t wg = warp >> 2, quarter = warp & 3;
        const uint32_t row = quarter * 32 + lane;                // row of this CTA == TMEM lane
        const uint32_t lane_addr = (quarter * 32) << 16;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        asm volatile("bar.sync 1, 256;" ::: "memory");           // the eight softmax warps
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            // this thread's half of its row -> columns 64 wg + 32 h .., two 16-bit elements per column
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const uint32_t chunk = wg * 16 + h * 8 + c;
                const uint4 x = *reinterpret_cast<const uint4 *>(p_s + row * (HD * 2) + ((chunk ^ (row & 7)) << 4));
                w[4 * c] = x.x; w[4 * c + 1] = x.y; w[4 * c + 2] = x.z; w[4 * c + 3] = x.w;
            }
            tmem_st32(tmem + lane_addr + kPairColQ + wg * 64 + h * 32, w);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_even(&sh->q_ready);

        const uint32_t s_addr = tmem + lane_addr + kPairColS;
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
        float m_own = -INFINITY, l_run = 0.f;                    // what this group's row sum is relative to (log2), and the sum
        bool ok = true;
        for (uint32_t j = wg; j < n_tiles; j += 2) {
            ok = warp_all(mbar_wait(&sh->s_full[wg], (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            uint32_t raw[4][32];
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) tmem_ld32(s_addr + c4 * 32, raw[c4]);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_even(&sh->s_read);        // the score tile may take the next product
            uint32_t bits[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
            if (form.masked(item, j)) form.visible(item, my_row0 + row, j, bits);
            if (__any_sync(0xffffffffu, (bits[0] & bits[1] & bits[2] & bits[3]) != 0xffffffffu)) {      // hidden keys become -inf before the (positive) scale
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4)
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(bits[c4] >> c & 1)) raw[c4][c] = 0xff800000u;
            }
            float mx4[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                mx4[x] = max3(__uint_as_float(raw[x][0]), __uint_as_float(raw[x][1]), __uint_as_float(raw[x][2]));
#pragma unroll
            for (int c = 3; c < 31; c += 2)
#pragma unroll
                for (int x = 0; x < 4; ++x) mx4[x] = max3(mx4[x], __uint_as_float(raw[x][c]), __uint_as_float(raw[x][c + 1]));
#pragma unroll
            for (int x = 0; x < 4; ++x) mx4[x] = fmaxf(mx4[x], __uint_as_float(raw[x][31]));
            const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * p.scale_log2;
            float m_prev = -INFINITY;
            if (j > 0) {
                ok = warp_all(mbar_wait(&sh->published[wg ^ 1][quarter], ((j - 1) >> 1) & 1));
                if (!ok) break;
                m_prev = sh->m_ref[wg ^ 1][row];
            }
            const float m_new = fmaxf(m_prev, mx);
            // keep the stale maximum while it is within 2^8 of the true one
            const bool raise = (m_new - m_prev > kRaiseThreshold) || (m_prev == -INFINITY && m_new != -INFINITY);
            const float m_cur = raise ? m_new : m_prev;
            sh->m_ref[wg][row] = m_cur;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->published[wg][quarter]);
            if (m_cur != m_own) {                                // raised here, or by the other group a tile ago
                l_run *= fast_exp2(m_own - m_cur);
                m_own = m_cur;
            }
            if (j > 1) {                                         // P.V of tile j-2 has left this group's P buffer
                ok = warp_all(mbar_wait(&sh->o_ready[wg], ((j - 2) >> 1) & 1));
                if (!ok) break;
            }
            if (j > 0 && __any_sync(0xffffffffu, raise)) {
                // O holds the sum over tiles < j; it may only be touched once P.V of tile j-1 has retired. P.V of tile j-3
                // has (the wait above), and P.V of tile j+1 cannot before this group's weights: the parity is unambiguous
                ok = warp_all(mbar_wait(&sh->o_ready[wg ^ 1], ((j - 1) >> 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const float factor = raise ? fast_exp2(m_prev - m_cur) : 1.f;    // exp2(-inf) == 0: the row of O was zero
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lane_addr + kPairColO + c0, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * factor);
                    tmem_st32(tmem + lane_addr + kPairColO + c0, o);
                }
                tmem_wait_st();
            }
            const float neg_m = (m_cur == -INFINITY) ? 0.f : -m_cur;
            const float2 shift2 = make_float2(neg_m, neg_m);
            float rs4[4] = {0.f, 0.f, 0.f, 0.f};
            unsigned char *prow = p_s + wg * kPairPBytes + row * 128;
#pragma unroll
            for (int c8 = 0; c8 < 16; ++c8) {                    // 8 keys: one 16-byte chunk of the P row
                uint32_t pk[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int at = (c8 & 3) * 8 + 2 * c;
                    const float2 x = fma2(make_float2(__uint_as_float(raw[c8 >> 2][at]), __uint_as_float(raw[c8 >> 2][at + 1])), scale2, shift2);
                    pk[c] = pack2<T>(fast_exp2(x.x), fast_exp2(x.y));   // P takes V's type: A and B of one tcgen05.mma share a format
                    rs4[c] = add_pair<T>(rs4[c], pk[c]);
                }
                *reinterpret_cast<uint4 *>(prow + (c8 >> 3) * 16384 + (((c8 & 7) ^ (row & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
            l_run += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            tc_fence_before();                      // orders a rescale of O before the P.V it precedes
            __syncwarp();
            if (lane == 0) mbar_arrive_even(&sh->p_ready[wg]);
        }

        // ---- the end: both groups, each with half of the head dims of every row ----
        const uint32_t last = n_tiles - 1, lw = last & 1;
        auto pair_sync = [&](uint32_t phase) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->pair[quarter]);
            return warp_all(mbar_wait(&sh->pair[quarter], phase));
        };
        if (ok && wg != lw) ok = warp_all(mbar_wait(&sh->published[lw][quarter], (last >> 1) & 1));
        if (ok) {
            const float m_fin = sh->m_ref[lw][row];
            if (m_fin != m_own) l_run *= fast_exp2(m_own - m_fin);
            m_own = m_fin;
            sh->l_sum[wg][row] = l_run;
        }
        // every arrival is made even after a failed wait, so that the partner does not run into its limit as well
        { const bool both = pair_sync(0); ok = ok && both; }
        // P.V of the last tile but one first: it retires after tile last-2, whose phase a parity could confuse with the last
        if (ok && n_tiles > 1) ok = warp_all(mbar_wait(&sh->o_ready[lw ^ 1], ((last - 1) >> 1) & 1));
        if (ok) ok = warp_all(mbar_wait(&sh->o_ready[lw], (last >> 1) & 1));
        if (ok) {
            tc_fence_after();
            const float l_tot = sh->l_sum[0][row] + sh->l_sum[1][row];
            const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;             // no visible key: zeros
            unsigned char *mine = ring + row * kPairStagePitch;            // all copies have landed, all products are done
#pragma unroll 1
            for (int c0 = 0; c0 < HD / 2; c0 += 32) {
                const int col = (int)wg * (HD / 2) + c0;
                uint32_t o[32];
                tmem_ld32(tmem + lane_addr + kPairColO + col, o);
                tmem_wait_ld();
                if constexpr (Form::kPartials) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4)
                        *reinterpret_cast<uint4 *>(mine + (col + c) * 4) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                } else {
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        uint4 v;
                        v.x = pack2<T>(__uint_as_float(o[c]) * inv, __uint_as_float(o[c + 1]) * inv);
                        v.y = pack2<T>(__uint_as_float(o[c + 2]) * inv, __uint_as_float(o[c + 3]) * inv);
                        v.z = pack2<T>(__uint_as_float(o[c + 4]) * inv, __uint_as_float(o[c + 5]) * inv);
                        v.w = pack2<T>(__uint_as_float(o[c + 6]) * inv, __uint_as_float(o[c + 7]) * inv);
                        *reinterpret_cast<uint4 *>(mine + (col + c) * 2) = v;
                    }
                }
            }
            if constexpr (Form::kPartials) {
                if (wg == 0 && form.exists(item, my_row0 + row)) {
                    const size_t prow = form.partial(item, my_row0 + row, ROWS);
                    form.part_m[prow] = m_own == -INFINITY ? -INFINITY : m_own * kLn2;   // natural-log domain
                    form.part_l[prow] = m_own == -INFINITY ? 0.f : l_tot;
                }
            }
        }
        { const bool both = pair_sync(1); ok = ok && both; }
        if (ok) {
            // whole rows: 16 of the quarter's 32 per warp
            constexpr uint32_t kRowBytes = Form::kPartials ? HD * 4 : HD * 2;
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t r = quarter * 32 + wg * 16 + i;
                if (!form.exists(item, my_row0 + r)) continue;
                unsigned char *dst;
                if constexpr (Form::kPartials) dst = reinterpret_cast<unsigned char *>(form.part_o + form.partial(item, my_row0 + r, ROWS) * HD);
                else dst = reinterpret_cast<unsigned char *>(form.output(item, my_row0 + r, HD));
#pragma unroll
                for (uint32_t b = lane * 16; b < kRowBytes; b += 512)
                    *reinterpret_cast<uint4 *>(dst + b) = *reinterpret_cast<const uint4 *>(ring + r * kPairStagePitch + b);
            }
        }
        failed = !ok;
    }

    if (failed) atomicOr(status, TT_DEV_WAIT_TIMEOUT);
    if (form.waits_late()) pdl_wait();
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();            // no product reads the other CTA's memory or TMEM any more
    if (warp == 8) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

template <typename T, class Form>
cudaError_t launch_pair(cudaStream_t stream, uint32_t n_items, const RowsParams &p, uint32_t *status, const Form &form) {
    auto kernel = attn_pair_kernel<T, Form>;
    cudaError_t e = tt_set_smem_once(kernel, kPairSmemBytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * n_items); cfg.blockDim = dim3(kPairThreads); cfg.dynamicSmemBytes = kPairSmemBytes; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tt_pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, p, status, form);
}

inline RowsParams pair_params(float scale, uint32_t io_dtype) {
    RowsParams p;
    p.scale_log2 = scale * kLog2e;
    const uint32_t m256 = (256u >> 4) << 24, m_mask = 31u << 24;
    p.idesc_qk = (tt_make_idesc_f16(io_dtype, 128, false) & ~m_mask) | m256;
    p.idesc_pv = (tt_make_idesc_f16(io_dtype, 256, true) & ~m_mask) | m256;
    return p;
}

}  // namespace
