// Attention of up to 128 query rows that share their keys, on the sm_100a tensor cores: the kernel behind the prefix
// pass of shared-prefix decode (attn_prefix.cu) and behind prefill with sinks (attn_prefill_sink.cu).
//
// A CTA takes an item: up to ROWS query rows of one KV head and a sequence of 128-key tiles. A row is a TMEM lane and
// one softmax thread per tile, so nothing of a row's softmax crosses threads:
//
//   S[j%2] = Q . K_j^T    SS MMA M128 N128 K16 x HD/16    TMEM columns 0..255, two score tiles
//   P_j    = exp2(S - m)  tcgen05.ld -> registers -> tcgen05.st over the first half of the tile's own columns
//   O     += P_j . V_j    TS MMA M128 N128 (N64 at head_dim 64) K16 x8 per 128 head dims     TMEM columns 256..
//
// Two softmax groups of ROWS/32 warps take the tiles in turn: while one group forms the weights of tile j, the other
// loads tile j+1 and takes its maxima, so the exponentials of one and the latencies of the other overlap, and the
// tensor pipe gets a tile of weights every half period. What the groups share is one number per row, the maximum m the
// weights of a tile are relative to: group j waits for m of tile j-1, decides m of tile j and publishes it before it
// starts on its exponentials. m is only raised when a score exceeds it by more than 2^8; the group that raises it
// rescales the row of O in TMEM (after P.V of tile j-1 has retired and before its own weights are handed over), and
// each group rescales its own row sum when it meets a raised m.
//
// Shared memory: Q and one ring of 16 KB slots that K and V chunks ([128 keys][64 head dims], 128-byte swizzle) travel
// through in the order the products consume them: K(0) K(1) V(0) K(2) V(1) ... At the end the ring's space takes the
// output tile, from which whole rows are stored.
//
// The softmax is 64 instructions of exp2 per row and 64 keys on a unit that does 16 a clock and SM, 1024 clocks a tile;
// the products are 2048 clocks at head_dim 256. Everything around the exponentials is therefore kept small: maxima three
// at a time, scale and shift as packed pairs, and the row sum straight from the packed 16-bit weights by adds that take
// one 16-bit and one 32-bit operand. Row sums are over the ROUNDED weights P.V uses, so O / l is a convex combination of
// V rows. Every mbarrier wait is bounded: a role whose wait runs out sets TT_DEV_WAIT_TIMEOUT and falls through to the
// common exit, where TMEM is released.
#pragma once

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

// A place in the ring of kSlots units, advanced without divisions: a producer that divides for every unit cannot keep up
// (measured on the pair kernel: 430 clocks a unit, 1700 of the 3100 clocks a tile took).
template <int SLOTS>
struct RingPos {
    uint32_t slot, lap;
    __device__ __forceinline__ explicit RingPos(uint32_t unit) : slot(unit % SLOTS), lap(unit / SLOTS) {}
    __device__ __forceinline__ void advance(uint32_t n) {      // n <= SLOTS
        slot += n;
        if (slot >= (uint32_t)SLOTS) { slot -= SLOTS; ++lap; }
    }
};
// Blocks of units in consumption order: K(0) | K(1) V(0) | K(2) V(1) | ... | V(n-1). First block of V, and how many blocks
// after its tile j the next one of its kind starts.
__device__ __forceinline__ uint32_t first_v_block(uint32_t n_tiles) { return n_tiles > 1 ? 2u : 1u; }
__device__ __forceinline__ uint32_t next_k_block(uint32_t j) { return j == 0 ? 1u : 2u; }
__device__ __forceinline__ uint32_t next_v_block(uint32_t j, uint32_t n_tiles) { return j + 2 < n_tiles ? 2u : 1u; }

// Warps: softmax group 0 from warp 0, group 1 from warp 4 (a warp may touch the TMEM lanes of its number modulo 4 alone);
// the K producer, the MMA warp and the V producer fill the numbers between and behind the groups.
template <int HD, int ROWS>
struct RowsGeom {
    static constexpr int kGroupWarps = ROWS / 32;
    static constexpr int kProducerWarp = ROWS == 128 ? 8 : 2, kMmaWarp = kProducerWarp + 1, kVProducerWarp = ROWS == 128 ? 10 : 6;
    static constexpr int kThreads = ROWS == 128 ? 352 : 224;
    static constexpr int kChunks = HD / 64;                     // ring units of one K or V tile
    static constexpr int kQSub = ROWS * 64 * 2;
    // the M = 128 products read rows ROWS..127 of the Q operand from what follows it in shared memory (their lanes are
    // never read), so the ring must follow Q directly; even, so that a pair of V chunks never wraps
    static constexpr int kSlots = ROWS == 64 || HD < 256 ? 12 : 10;
    static constexpr int kOffRing = kQSub * kChunks;
    static constexpr int kOffMisc = kOffRing + kSlots * kSlotBytes;
    static constexpr int kStagePitch = HD * 4 + 16;             // bytes; 16-byte accesses of 8 lanes meet 8 bank groups
    static_assert(ROWS * kStagePitch <= kSlots * kSlotBytes, "the output tile must fit the ring");
};

struct RowsShared {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t q_ready;           // one arrive per softmax warp: Q is in shared memory
    uint64_t s_full[2];
    uint64_t p_ready[2];        // one arrive per warp of the group
    uint64_t o_ready[2];        // [tile parity]: P.V of the tile has retired
    uint64_t published[2][4];   // [tile parity][lane quarter]: m of the tile is in m_ref
    uint64_t pair[4];           // the two warps of a lane quarter, at the end
    float l_sum[2][128];        // the groups' row sums, at the end
    float m_ref[2][128];
    uint32_t tmem_base;
    uint32_t pad;
};
template <int HD, int ROWS>
constexpr int rows_smem_bytes() { return RowsGeom<HD, ROWS>::kOffMisc + (int)sizeof(RowsShared); }
static_assert(rows_smem_bytes<256, 128>() <= 232448 && rows_smem_bytes<256, 64>() <= 232448 && rows_smem_bytes<128, 128>() <= 232448,
              "shared memory exceeds the per-CTA limit");

// What an item is, the same for every form.
struct RowsItem {
    uint32_t kv_head, n_tiles;
    uint32_t n_halves;                   // halves of 64 keys in use: the last tile may have one
};

// bits lo .. hi-1 of a word's 32, for any lo and hi
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
    const uint32_t below_hi = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u;
    const uint32_t below_lo = lo >= 32 ? 0xffffffffu : lo <= 0 ? 0u : (1u << lo) - 1u;
    return below_hi & ~below_lo;
}

struct RowsParams {
    float scale_log2;
    uint32_t idesc_qk, idesc_pv;
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// sum + both halves of a packed pair of 16-bit numbers, each add with one 16-bit operand
template <typename T>
__device__ __forceinline__ float add_pair(float sum, uint32_t packed);
template <>
__device__ __forceinline__ float add_pair<__half>(float sum, uint32_t packed) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tadd.rn.f32.f16 %0, lo, %0;\n\tadd.rn.f32.f16 %0, hi, %0;\n\t}"
        : "+f"(sum) : "r"(packed));
    return sum;
}
template <>
__device__ __forceinline__ float add_pair<__nv_bfloat16>(float sum, uint32_t packed) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tadd.rn.f32.bf16 %0, lo, %0;\n\tadd.rn.f32.bf16 %0, hi, %0;\n\t}"
        : "+f"(sum) : "r"(packed));
    return sum;
}

// Issues the asynchronous copies of query rows row0 + first, row0 + first + step, ... (N of them) of a CTA by one warp, 16
// bytes a lane; `at(r, chunk)` is where chunk `chunk` of the CTA's row r goes. Rows that do not exist become zeros.
template <int HD, int ROWS, int N, class Form, class At>
__device__ __forceinline__ void load_query_rows(const Form &form, const typename Form::Item &item, uint32_t row0, uint32_t first,
                                                uint32_t step, uint32_t lane, At at) {
    static_assert(N <= 32, "one lane looks a row up");
    constexpr uint32_t kLanes = HD / 8, kAtOnce = 32 / kLanes;       // lanes a row takes, rows per round
    // the rows' addresses, one per lane: a lookup may be a search
    const unsigned long long mine = lane < (uint32_t)N ? (unsigned long long)form.query(item, row0 + first + lane * step, HD, ROWS) : 0ull;
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)N; i += kAtOnce) {
        const uint32_t nth = i + lane / kLanes, r = first + nth * step, chunk = lane % kLanes;
        const unsigned char *src = (const unsigned char *)__shfl_sync(0xffffffffu, mine, nth);
        unsigned char *dst = at(r, chunk);
        if (src != nullptr)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src + chunk * 16) : "memory");
        else
            *reinterpret_cast<uint4 *>(dst) = make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// A Form says what the items are. It provides
//   struct Item : RowsItem
//   Item item(block, HD, ROWS)                 from the block index and the parameters (or tables that a copy, not a kernel,
//                                              brought: it runs ahead of the wait for the kernel before)
//   const void *query(item, row, HD, ROWS)     start of a row's query (null: no such row)
//   void acquire(item)                         one thread, before its first load: fences the tensor maps if they need it
//   const CUtensorMap *box(item, tile, half, is_k, row)   keys 64 half .. of a tile: the map (boxes [64 rows][64]), the row
//   bool masked(item, tile)                    whether some row of the item does not see all 128 keys of the tile
//   void visible(item, row, tile, bits)        bit c % 32 of bits[c / 32]: key c of the tile is visible to the row
//   bool exists(item, row)
//   kPartials                                  true: (m, l, o) partial rows; false: normalised rows of T
//   partial(item, row, HD) / output(item, row, HD)     partial row number / where the row goes
//   float *part_o, *part_m, *part_l            (kPartials)
//   bool waits_late()                          the launch before this one produces nothing it reads and has waited for those
//                                              that do: a CTA waits for its end only before it ends itself
template <typename T, int HD, int ROWS, class Form>
__global__ void __launch_bounds__(RowsGeom<HD, ROWS>::kThreads, 1)
attn_rows_kernel(RowsParams p, uint32_t *__restrict__ status, const __grid_constant__ Form form) {
    using G = RowsGeom<HD, ROWS>;
    constexpr int kSlots = G::kSlots, kQSub = G::kQSub, kChunks = G::kChunks;
    // nearly every byte is spoken for, so there is no slack to align the tiles by hand: the dynamic window of a kernel
    // without static shared memory starts 1024-byte aligned, and a launch where it does not is refused rather than run
    // with broken swizzles
    extern __shared__ __align__(1024) unsigned char smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(status, TT_DEV_BAD_ITEM);
        return;
    }
    unsigned char *q_s = smem;
    unsigned char *ring = smem + G::kOffRing;
    RowsShared *sh = reinterpret_cast<RowsShared *>(smem + G::kOffMisc);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_launch_dependents();
    const typename Form::Item item = form.item(blockIdx.x, HD, ROWS);        // from the parameters alone
    if (!form.waits_late()) pdl_wait();       // the kernel before this one may have produced the query or cache rows
    const uint32_t n_tiles = item.n_tiles;                                   // >= 1

    // the producers: block after block of K's (or V's) units, each into its place of the ring once that is free
    auto produce = [&](bool is_k) {
        RingPos<kSlots> pos(is_k ? 0u : first_v_block(n_tiles) * kChunks);
        const uint32_t x0 = item.kv_head * HD;
        uint32_t issued = 0;
        bool ok = true;
        for (uint32_t j = 0; j < n_tiles; ++j) {
            int row[2];
            const CUtensorMap *map[2];
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) map[half] = form.box(item, j, half, is_k, row[half]);
#pragma unroll 1
            for (uint32_t c = 0; c < (uint32_t)kChunks; ++c) {
                if (pos.lap > 0) ok = mbar_wait(&sh->empty[pos.slot], (pos.lap - 1) & 1);
                if (!ok) break;
                uint64_t *bar = &sh->full[pos.slot];
                unsigned char *dst = ring + pos.slot * kSlotBytes;
                mbar_expect_tx(bar, kSlotBytes);
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                    tma_load_2d(dst + half * (kSlotBytes / 2), map[half], (int)(x0 + c * 64), row[half], bar);
                ++issued;
                pos.advance(1);
            }
            if (!ok) break;
            pos.advance(((is_k ? next_k_block(j) : next_v_block(j, n_tiles)) - 1) * kChunks);
        }
        if (!ok) {
            // give this thread's copies still in flight a bounded chance to land before the shared memory is released
            RingPos<kSlots> p2(is_k ? 0u : first_v_block(n_tiles) * kChunks);
            for (uint32_t j = 0, n = 0; n < issued; ++j) {
                for (uint32_t c = 0; c < (uint32_t)kChunks && n < issued; ++c, ++n) {
                    if (n + kSlots >= issued) mbar_wait(&sh->full[p2.slot], p2.lap & 1, 1u << 16);
                    p2.advance(1);
                }
                p2.advance(((is_k ? next_k_block(j) : next_v_block(j, n_tiles)) - 1) * kChunks);
            }
        }
        return ok;
    };
    if (threadIdx.x == G::kProducerWarp * 32) {
        for (int s = 0; s < kSlots; ++s) { mbar_init(&sh->full[s], 1); mbar_init(&sh->empty[s], 1); }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sh->s_full[s], 1);
            mbar_init(&sh->p_ready[s], G::kGroupWarps);
            mbar_init(&sh->o_ready[s], 1);
            for (int w = 0; w < 4; ++w) mbar_init(&sh->published[s][w], 1);
        }
        for (int w = 0; w < 4; ++w) mbar_init(&sh->pair[w], 2);
        mbar_init(&sh->q_ready, 2 * G::kGroupWarps);
        mbar_fence_init();
    }
    if (warp != G::kProducerWarp && warp != G::kMmaWarp && warp != G::kVProducerWarp)
        // Q: K-major, 128-byte swizzle, 64-wide sub-tiles; in flight while the barriers and TMEM are set up
        load_query_rows<HD, ROWS, ROWS / (2 * G::kGroupWarps)>(form, item, 0, (warp >> 2) * G::kGroupWarps + (warp & 3), 2 * G::kGroupWarps, lane,
                                                               [&](uint32_t r, uint32_t chunk) {
            return q_s + (chunk >> 3) * kQSub + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
        });
    if (warp == G::kProducerWarp) {
        __syncwarp();
        tmem_alloc(&sh->tmem_base, kTmemCols);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    bool failed = false;

    if (warp == G::kProducerWarp || warp == G::kVProducerWarp) {
        // ------------------------------------------------------------------ TMA producers: K, V
        if (lane == 0) {
            form.acquire(item);
            failed = !produce(warp == G::kProducerWarp);
        }
    } else if (warp == G::kMmaWarp) {
        // ------------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            const uint32_t ring_a = smem_u32(ring), q_a = smem_u32(q_s);
            RingPos<kSlots> pos(0);            // units are consumed in the order of the ring
            auto issue_qk = [&](uint32_t j) {
                const uint32_t d = tmem + kColS + (j & 1) * kBK;
#pragma unroll 1
                for (uint32_t c = 0; c < (uint32_t)kChunks; ++c, pos.advance(1)) {
                    const uint32_t slot = pos.slot;
                    if (!mbar_wait(&sh->full[slot], pos.lap & 1)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {
                        const uint64_t ad = make_desc(q_a + c * kQSub + ks * 32, 16, 1024);
                        const uint64_t bd = make_desc(ring_a + slot * kSlotBytes + ks * 32, 16, 1024);
                        mma_ss(d, ad, bd, p.idesc_qk, (c > 0 || ks > 0) ? 1u : 0u);
                    }
                    mma_commit(&sh->empty[slot]);
                }
                mma_commit(&sh->s_full[j & 1]);
                return true;
            };
            bool ok = mbar_wait(&sh->q_ready, 0);
            tc_fence_after();
            if (ok) ok = issue_qk(0);
            for (uint32_t j = 0; ok && j < n_tiles; ++j) {
                // S of tile j+1 goes where P of tile j-1 is read from: that product was issued before this one
                if (j + 1 < n_tiles) ok = issue_qk(j + 1);
                if (ok) ok = mbar_wait(&sh->p_ready[j & 1], (j >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t p_t = tmem + kColS + (j & 1) * kBK;    // P_j: 64 columns of 16-bit pairs over S_j
                // O(128 head dims) += P_j . V_j: V as the MN-major B operand, 64-wide head-dim atoms one slot apart
                // (LBO), 8-key groups 1024 B apart (SBO), 16 keys (2048 B) per step
                constexpr uint32_t kUnits = kChunks == 1 ? 1 : 2;      // ring units per product
                for (uint32_t c = 0; ok && c < (uint32_t)kChunks; c += kUnits, pos.advance(kUnits)) {
                    const uint32_t slot = pos.slot;
                    for (uint32_t x = 0; ok && x < kUnits; ++x) ok = mbar_wait(&sh->full[slot + x], pos.lap & 1);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; ++kk) {
                        const uint64_t bd = make_desc(ring_a + slot * kSlotBytes + kk * 2048, kSlotBytes, 1024);
                        mma_ts(tmem + kColO + c * 64, p_t + kk * 8, bd, p.idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                    }
                    for (uint32_t x = 0; x < kUnits; ++x) mma_commit(&sh->empty[slot + x]);
                }
                if (!ok) break;
                mma_commit(&sh->o_ready[j & 1]);
            }
            failed = !ok;
        }
    } else {
        // ------------------------------------------------------------------ softmax: group `wg` takes tiles wg, wg + 2, ...
        const uint32_t wg = warp >= 4 ? 1u : 0u, quarter = warp & 3;
        const uint32_t row = quarter * 32 + lane;                // row of the item == TMEM lane
        const uint32_t lane_addr = (quarter * 32) << 16;
        const uint32_t s_addr = tmem + lane_addr + kColS + wg * kBK;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_ready);
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
            uint32_t bits[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
            if (form.masked(item, j)) form.visible(item, row, j, bits);
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
            if (j > 0 && __any_sync(0xffffffffu, raise)) {
                // O holds the sum over tiles < j; it may only be touched once P.V of tile j-1 has retired
                ok = warp_all(mbar_wait(&sh->o_ready[wg ^ 1], ((j - 1) >> 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const float factor = raise ? fast_exp2(m_prev - m_cur) : 1.f;    // exp2(-inf) == 0: the row of O was zero
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
            const float neg_m = (m_cur == -INFINITY) ? 0.f : -m_cur;
            const float2 shift2 = make_float2(neg_m, neg_m);
            float rs4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c4 = 0; c4 < 4; ++c4) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float2 x = fma2(make_float2(__uint_as_float(raw[c4][2 * c]), __uint_as_float(raw[c4][2 * c + 1])), scale2, shift2);
                    pk[c] = pack2<T>(fast_exp2(x.x), fast_exp2(x.y));   // P takes V's type: A and B of one tcgen05.mma share a format
                    rs4[c & 3] = add_pair<T>(rs4[c & 3], pk[c]);
                }
                tmem_st16(s_addr + c4 * 16, pk);    // over columns of this score tile that have been read above
            }
            l_run += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
            tmem_wait_st();
            tc_fence_before();                      // orders P and a rescale of O before the P.V they precede
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->p_ready[wg]);
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
        // P.V of the last tile but one first: a barrier's parity cannot tell its phase from the one before the last
        if (ok && n_tiles > 1) ok = warp_all(mbar_wait(&sh->o_ready[lw ^ 1], ((last - 1) >> 1) & 1));
        if (ok) ok = warp_all(mbar_wait(&sh->o_ready[lw], (last >> 1) & 1));
        if (ok) {
            tc_fence_after();
            const float l_tot = sh->l_sum[0][row] + sh->l_sum[1][row];
            const float inv = l_tot > 0.f ? 1.f / l_tot : 0.f;             // no visible key: zeros
            unsigned char *mine = ring + row * G::kStagePitch;             // all copies have landed, all products are done
#pragma unroll 1
            for (int c0 = 0; c0 < HD / 2; c0 += 32) {
                const int col = (int)wg * (HD / 2) + c0;
                uint32_t o[32];
                tmem_ld32(tmem + lane_addr + kColO + col, o);
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
                if (wg == 0 && form.exists(item, row)) {
                    const size_t prow = form.partial(item, row, ROWS);
                    form.part_m[prow] = m_own == -INFINITY ? -INFINITY : m_own * kLn2;   // natural-log domain
                    form.part_l[prow] = m_own == -INFINITY ? 0.f : l_tot;
                }
            }
        }
        { const bool both = pair_sync(1); ok = ok && both; }
        if (ok) {
            // whole rows: 16 of the quarter's 32 per warp
            constexpr uint32_t kRowBytes = Form::kPartials ? HD * 4 : HD * 2, kLanes = kRowBytes / 16 < 32 ? kRowBytes / 16 : 32;
            constexpr uint32_t kAtOnce = 32 / kLanes;
            for (uint32_t i = 0; i < 16; i += kAtOnce) {
                const uint32_t r = quarter * 32 + wg * 16 + i + lane / kLanes;
                if (!form.exists(item, r)) continue;
                unsigned char *dst;
                if constexpr (Form::kPartials) dst = reinterpret_cast<unsigned char *>(form.part_o + form.partial(item, r, ROWS) * HD);
                else dst = reinterpret_cast<unsigned char *>(form.output(item, r, HD));
#pragma unroll
                for (uint32_t b = (lane % kLanes) * 16; b < kRowBytes; b += kLanes * 16)
                    *reinterpret_cast<uint4 *>(dst + b) = *reinterpret_cast<const uint4 *>(ring + r * G::kStagePitch + b);
            }
        }
        failed = !ok;
    }

    if (failed) atomicOr(status, TT_DEV_WAIT_TIMEOUT);
    if (form.waits_late()) pdl_wait();
    tc_fence_before();
    __syncthreads();
    if (warp == G::kProducerWarp) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <typename T, int HD, int ROWS, class Form>
cudaError_t launch_rows(cudaStream_t stream, uint32_t n_items, const RowsParams &p, uint32_t *status, const Form &form) {
    auto kernel = attn_rows_kernel<T, HD, ROWS, Form>;
    const int smem = rows_smem_bytes<HD, ROWS>();
    cudaError_t e = tt_set_smem_once(kernel, smem);
    if (e != cudaSuccess) return e;
    return tt_launch_pdl(kernel, dim3(n_items), dim3(RowsGeom<HD, ROWS>::kThreads), (size_t)smem, stream, p, status, form);
}

inline RowsParams rows_params(float scale, uint32_t io_dtype, uint32_t head_dim) {
    RowsParams p;
    p.scale_log2 = scale * kLog2e;
    p.idesc_qk = tt_make_idesc_f16(io_dtype, kBK, false);                           // Q (K-major) x K rows (K-major)
    p.idesc_pv = tt_make_idesc_f16(io_dtype, head_dim == 64 ? 64 : 128, true);      // P (TMEM) x V (MN-major)
    return p;
}

}  // namespace
