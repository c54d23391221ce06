// Pass 1 of the split-KV decode attention (mma.sync): the kernel, in the forms its callers instantiate.
#pragma once

#include "tt_sm100.h"

namespace {

constexpr int kKeysPerBlock = 16;   // keys per warp pipeline stage
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1);

template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4],
                                                  uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                         uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A store whose lines are the last to leave L2: read back by the next launch, next to a stream of K and V that is not
// (scores of 435,000 keys: 216.5 -> 212.7 us a call).
__device__ __forceinline__ void store_keep(float *dst, float x, float y) {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    asm volatile("st.global.L2::cache_hint.v2.f32 [%0], {%1, %2}, %3;" ::"l"(dst), "f"(x), "f"(y), "l"(policy) : "memory");
}

// Shared memory of the fp16/bf16 pass-1 kernel for HPC KV heads per CTA.
template <int HD, int HPC>
struct DecodeSmem {
    static constexpr int kPitch = HPC * HD + 8;                    // elements per staged row (all HPC heads of a key)
    static constexpr int kRowBytes = kPitch * 2;
    static constexpr int kTileBytes = kKeysPerBlock * kRowBytes;   // one K (or V) block
    static constexpr int kVRing = kStages * kTileBytes;            // K ring first, V ring behind it
    static constexpr int kRingBytes = 2 * kStages * kTileBytes;
    static constexpr int kScorePitch = 24;                         // floats per query row of a handed-over score tile
    static constexpr int kScoreTile = 16 * kScorePitch;            // [query row][key]
    static constexpr int kScoreBytes = HPC * 2 * kScoreTile * 4;   // [head][buffer]
    static constexpr int kBars = 4 * kStages + 4 * HPC;            // k_full, v_full, k_empty, v_empty [kStages]; s_full, s_empty [HPC][2]
    static constexpr int kTotal = kRingBytes + kScoreBytes + kBars * 8;
};

// The forms of pass 1. What a form needs beyond the plain kernel travels in its PassExtra.
//   kPassSink    the keys of a session are its first `sink` keys and the union of its rows' sliding
//                windows behind them, addressed by a compact index c: key = c for c < sink, else
//                kv_start + c - sink (kv_start = first key of that union, never below sink). Row r sees
//                key < sink or key + window >= end_r. In a ring cache of R rows behind the sinks, key >=
//                sink lives at row sink + (key - sink) % R.
//   kPassScores  besides the partials, the raw scores q.k go to ses.scores[kv head][key][packed row] and
//                each row's (max, sum) of the item in log2 units with UNROUNDED weights to part_m2 / part_l2,
//                from which the weights of the whole softmax are formed once every part is done.
//   kPassSinkCluster   kPassSink whose parts of a (session, KV heads, row tile) are the CTAs of one cluster: they
//                leave (m, l, O) in their shared memory, and each forms a slice of the output columns from all
//                of them. No partials, no second launch.
enum : int { kPassPlain = 0, kPassSink = 1, kPassScores = 2, kPassSinkCluster = 3 };
constexpr uint32_t kMaxSinkCluster = 16;
template <int FORM>
struct PassExtra {
    // the next launch may start once every CTA has seen the end of the launches before this one; it then need not wait
    // for this one's results before it reads what they left
    uint32_t dependents_late;
};
template <>
struct PassExtra<kPassSink> { uint32_t sink, window; };
template <>
struct PassExtra<kPassSinkCluster> {
    uint32_t sink, window, cluster, out_row_stride;
    int *resident;               // host: launch nothing, store how many clusters run at once
};
template <>
struct PassExtra<kPassScores> { float *part_m2, *part_l2; };

// ---------------------------------------------------------------------------------------
// Pass 1. grid = items, block = 2 * HPC warps; 4 / HPC CTAs per SM.
//
// A work item is (session, HPC adjacent KV heads, up to 16 packed query rows per head, key range).
// With HPC = 2 a CTA streams whole cache rows (both KV heads of a key, 1 KB at head_dim 256) so
// that DRAM is read in long contiguous pieces; a pure streaming read of 512-byte pieces at a 1 KB
// pitch measured 6.6 TB/s on this part against 7.1 TB/s for whole rows.
//
// The warps of a CTA have different jobs and run one block apart. Both products are TRANSPOSED so
// that the 8-wide N dimension of mma.m16n8k16 is the query rows of one KV head (8 with a GQA group
// of 8, two n-tiles for up to 16 packed rows) and the 16-wide M dimension is filled by keys
// (Q.K^T) or head dimensions (P.V) -- nothing is padding:
//   warps 0 .. HPC-1      (one per KV head) form S^T = K . Q^T from the K ring (A = the K block read
//                         with ldmatrix, B = the query rows held in registers) and hand the
//                         16 x 8 score tile over through shared memory;
//   warps HPC .. 2 HPC-1  take the score tile in the B-operand layout (one query row per lane
//                         quad-row, so a row's maximum is two shuffles), run the online softmax
//                         and accumulate O^T += V^T . P^T from the V ring (A = the V block read
//                         with ldmatrix.trans); they end with (m, l) and the whole output tile.
// K and V have their own 3-stage rings of bulk copies (one per key row, completion on the stage's
// mbarrier). Warp 0 refills a K stage once every K.Q^T warp has released it, warp HPC a V stage
// once every P.V warp has; the score tiles are double buffered per head. Every wait is bounded.
// ---------------------------------------------------------------------------------------
template <int HD, int NT, int HPC, typename T, int FORM>
__global__ void __launch_bounds__(64 * HPC, 4 / HPC)
attn_decode_partial_kernel(const TTDecodeItem *__restrict__ items,
                           const TTDecodeSession *__restrict__ sessions, float *__restrict__ part_o,
                           float *__restrict__ part_m, float *__restrict__ part_l,
                           uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t kv_stride_bytes,
                           uint32_t q_row_stride, float scale_log2, uint32_t *__restrict__ status,
                           const __grid_constant__ TTSessionTable table, uint32_t table_keys_per_item,
                           PassExtra<FORM> extra) {
    using S = DecodeSmem<HD, HPC>;
    constexpr bool SINK = FORM == kPassSink || FORM == kPassSinkCluster;
    constexpr int KS = HD / 16;         // k-steps of K.Q^T and m-tiles of V^T.P^T
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int role = warp / HPC, head = warp % HPC;   // role 0: K.Q^T, role 1: softmax + V^T.P^T

    const uint32_t group = n_q_heads / n_kv_heads;
    const uint32_t n_kv_groups = n_kv_heads / HPC;
    // Calls with up to kParamSessions sessions carry them in the kernel parameters and derive the
    // work item from the block index (the items of a session are equal slices, item_prefix says
    // where each session's items start), so no table is copied to the device and a CTA starts
    // without two dependent global loads.
    bool dependents_late = false;
    if constexpr (FORM == kPassPlain) dependents_late = extra.dependents_late != 0;
    if (!dependents_late) pdl_launch_dependents();
    TTDecodeItem item;
    TTDecodeSession ses;
    if (table.n != 0) {
        uint32_t lo = 0, hi = table.n;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (table.item_prefix[mid] <= blockIdx.x) lo = mid; else hi = mid;
        }
        ses = table.s[lo];
        const uint32_t local = blockIdx.x - table.item_prefix[lo];
        const uint32_t packed_rows = ses.q_rows * group;
        const uint32_t row_tiles = (packed_rows + 15) / 16;
        uint32_t unit = local, part = 0;
        if constexpr (FORM == kPassSinkCluster) { part = local % extra.cluster; unit = local / extra.cluster; }
        const uint32_t rt = unit % row_tiles, kvg = (unit / row_tiles) % n_kv_groups;
        if constexpr (FORM != kPassSinkCluster) part = local / (row_tiles * n_kv_groups);
        item.session = lo; item.kv_head = kvg * HPC; item.part_index = part; item.partial_base = ses.partial_base;
        if constexpr (SINK) {
            const uint32_t visible = min(extra.sink, ses.seq_len) + (ses.seq_len > ses.kv_start ? ses.seq_len - ses.kv_start : 0u);
            uint32_t keys = table_keys_per_item;
            if constexpr (FORM == kPassSinkCluster) {      // a cluster's own keys, in whole blocks
                keys = (visible + extra.cluster - 1) / extra.cluster;
                keys = (keys + kKeysPerBlock - 1) / kKeysPerBlock * kKeysPerBlock;
            }
            item.key_begin = min(visible, part * keys);
            item.key_end = min(visible, item.key_begin + keys);
        } else {
            item.key_begin = min(ses.seq_len, ses.kv_start + part * table_keys_per_item);
            item.key_end = min(ses.seq_len, item.key_begin + table_keys_per_item);
        }
        item.row_begin = rt * 16;
        item.row_count = min(16u, packed_rows - rt * 16);
    } else {
        item = items[blockIdx.x];
        ses = sessions[item.session];
    }
    const uint32_t kv_head = item.kv_head + head;      // the head this warp serves

    unsigned char *k_ring = smem;
    unsigned char *v_ring = smem + S::kVRing;
    float *score = reinterpret_cast<float *>(smem + S::kRingBytes) + head * 2 * S::kScoreTile;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kRingBytes + S::kScoreBytes);
    uint64_t *k_full = bars, *v_full = bars + kStages, *k_empty = bars + 2 * kStages, *v_empty = bars + 3 * kStages;
    uint64_t *s_full = bars + 4 * kStages + head * 4, *s_empty = s_full + 2;

    if (threadIdx.x == 0) {
        for (int b = 0; b < 2 * kStages; ++b) mbar_init(&bars[b], 1);                   // filled by one expect_tx arrival
        for (int b = 2 * kStages; b < 4 * kStages; ++b) mbar_init(&bars[b], HPC);       // released by every reader warp
        for (int b = 4 * kStages; b < S::kBars; ++b) mbar_init(&bars[b], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // everything above overlapped the tail of the kernel before this one in the stream; its
    // results (the query rows, the newest K/V rows, partials being merged) are read from here on
    pdl_wait();
    if (dependents_late) pdl_launch_dependents();

    const uint32_t n_keys = item.key_end - item.key_begin;
    const uint32_t n_blocks = (n_keys + kKeysPerBlock - 1) / kKeysPerBlock;
    auto block_valid = [&](uint32_t i) { return min((uint32_t)kKeysPerBlock, n_keys - i * kKeysPerBlock); };
    // lanes 0..15 of the issuing warp fetch one row each (all HPC heads of the key) of block i
    auto issue = [&](uint32_t i, unsigned char *ring, const unsigned char *base, uint64_t *full, bool zero_fill) {
        const uint32_t valid = block_valid(i), stage = i % kStages;
        if (lane == 0) mbar_expect_tx(&full[stage], valid * (uint32_t)(HPC * HD * 2));
        __syncwarp();
        if (lane < kKeysPerBlock) {
            unsigned char *dst = ring + stage * S::kTileBytes + lane * S::kRowBytes;
            if ((uint32_t)lane < valid) {
                uint32_t p = item.key_begin + i * kKeysPerBlock + lane;
                if constexpr (SINK) {
                    if (p >= extra.sink) {
                        p = ses.kv_start + (p - extra.sink);
                        if (ses.ring_capacity) p = extra.sink + (p - extra.sink) % ses.ring_capacity;
                    }
                } else if constexpr (FORM == kPassPlain) {
                    if (ses.row_index != nullptr) p = ses.row_index[p];
                    if (ses.ring_capacity) p %= ses.ring_capacity;
                }
                // read once: evict-first in L2, so that the stream does not push out the partials, the query
                // rows and what the neighbouring kernels of the step keep there (measured on the config-2
                // step: 0.1854 -> 0.1778 ms)
                bulk_copy_g2s_stream(dst, base + (size_t)p * kv_stride_bytes, HPC * HD * 2, &full[stage]);
            } else if (zero_fill) {
                // a V row that is never fetched must still be finite: it meets p == 0 in P.V
                const uint4 z = make_uint4(0u, 0u, 0u, 0u);
                for (int c = 0; c < HPC * HD / 8; ++c) reinterpret_cast<uint4 *>(dst)[c] = z;
            }
        }
    };
    bool timed_out = false;
    uint32_t consumed = 0, issued = 0;      // blocks of the ring this warp fills (warps 0 and HPC only)

    if (role == 0) {
        // ================= K . Q^T =================
        const unsigned char *kbase = reinterpret_cast<const unsigned char *>(ses.k) + (size_t)item.kv_head * HD * 2;
        // the query rows as B fragments: lane (g, t) holds dims 2t, 2t+1 (+8) of row g of every n-tile
        uint32_t qf[NT][KS][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t r = nt * 8 + g;
            const T *qp = nullptr;
            if (r < item.row_count) {
                const uint32_t packed = item.row_begin + r;
                qp = reinterpret_cast<const T *>(ses.q) + (size_t)(packed / group) * q_row_stride +
                     (size_t)(kv_head * group + packed % group) * HD + t * 2;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                qf[nt][ks][0] = qp ? *reinterpret_cast<const uint32_t *>(qp + ks * 16) : 0u;
                qf[nt][ks][1] = qp ? *reinterpret_cast<const uint32_t *>(qp + ks * 16 + 8) : 0u;
            }
        }
        if (head == 0)
            for (; issued < n_blocks && issued < (uint32_t)kStages; ++issued) issue(issued, k_ring, kbase, k_full, false);
        // A fragment of a K block: matrix j = lane / 8 covers keys 8 (j & 1) .. +7, dims 8 (j >> 1) .. +7
        const uint32_t k_off = ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kRowBytes + (lane >> 4) * 16 + head * HD * 2;
        for (uint32_t i = 0; i < n_blocks; ++i) {
            if (!warp_all(mbar_wait(&k_full[i % kStages], (i / kStages) & 1))) { timed_out = true; break; }
            const uint32_t stage = smem_u32(k_ring + (i % kStages) * S::kTileBytes);
            // two accumulator chains per n-tile (even / odd k-steps) halve the dependent MMA depth
            float s0[NT][4], s1[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) { s0[nt][0] = s0[nt][1] = s0[nt][2] = s0[nt][3] = 0.f; s1[nt][0] = s1[nt][1] = s1[nt][2] = s1[nt][3] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < KS; ks += 2) {
                uint32_t a[4], b[4];
                ldmatrix_x4(a, stage + k_off + ks * 32);
                ldmatrix_x4(b, stage + k_off + (ks + 1) * 32);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_16816<T>(s0[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
                    mma_16816<T>(s1[nt], b, qf[nt][ks + 1][0], qf[nt][ks + 1][1]);
                }
            }
            __syncwarp();                                   // every lane has its fragments: this warp releases the stage
            if (lane == 0) mbar_arrive(&k_empty[i % kStages]);
            if (head == 0) consumed = i + 1;
            // hand the tile over: element (query row r, key k) at score[buffer][r][k]
            if (i >= 2 && !warp_all(mbar_wait(&s_empty[i & 1], ((i >> 1) - 1) & 1))) { timed_out = true; break; }
            float *sb = score + (i & 1) * S::kScoreTile;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float *r0 = sb + (nt * 8 + 2 * t) * S::kScorePitch, *r1 = r0 + S::kScorePitch;
                r0[g] = s0[nt][0] + s1[nt][0]; r1[g] = s0[nt][1] + s1[nt][1];
                r0[g + 8] = s0[nt][2] + s1[nt][2]; r1[g + 8] = s0[nt][3] + s1[nt][3];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_full[i & 1]);
            if (head == 0 && issued < n_blocks) {           // block i + kStages goes into the stage block i just left
                if (!warp_all(mbar_wait(&k_empty[i % kStages], (i / kStages) & 1))) { timed_out = true; break; }
                issue(issued, k_ring, kbase, k_full, false);
                ++issued;
            }
            if constexpr (FORM == kPassScores) {
                // behind the refill, which must not wait for them; 8 keys x 8 rows per store: 256 contiguous bytes of the warp when the row count is padded to 8
                const uint32_t rows_pad = (ses.q_rows * group + 8 * NT - 1) / (8 * NT) * (8 * NT);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (nt * 8 + 2 * t >= item.row_count) continue;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t key = item.key_begin + i * kKeysPerBlock + g + 8 * h;
                        if (key < item.key_end)
                            store_keep(ses.scores + ((size_t)kv_head * ses.seq_len + key) * rows_pad + item.row_begin + nt * 8 + 2 * t,
                                       s0[nt][2 * h] + s1[nt][2 * h], s0[nt][2 * h + 1] + s1[nt][2 * h + 1]);
                    }
                }
            }
        }
        if (timed_out) {
            // blocks issued into the ring and not yet waited for may still be landing
            for (uint32_t b = consumed; b < issued; ++b) mbar_wait(&k_full[b % kStages], (b / kStages) & 1, 1u << 16);
            if (lane == 0) atomicOr(status, TT_DEV_WAIT_TIMEOUT);
        }
        return;
    }

    // ================= softmax and V^T . P^T =================
    const unsigned char *vbase = reinterpret_cast<const unsigned char *>(ses.v) + (size_t)item.kv_head * HD * 2;
    if (head == 0)
        for (; issued < n_blocks && issued < (uint32_t)kStages; ++issued) issue(issued, v_ring, vbase, v_full, true);

    float acc[NT][KS][4];               // O^T: dims 16 mt + g (+8) x query rows 2t, 2t+1 of n-tile nt
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) acc[nt][mt][0] = acc[nt][mt][1] = acc[nt][mt][2] = acc[nt][mt][3] = 0.f;
    float m_run[NT], l_run[NT];         // of query row 8 nt + g; l is this lane's share (keys 2t, 2t+1, 2t+8, 2t+9)
    float l_true[NT];                   // kPassScores: the same sum over the unrounded weights
    uint32_t limit[NT];                 // visible-key limit of that row
    const uint32_t w_first = item.row_begin / group;
    const uint32_t limit_min = ses.seq_len - (ses.q_rows - 1 - w_first);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m_run[nt] = -INFINITY; l_run[nt] = 0.f; l_true[nt] = 0.f;
        const uint32_t r = nt * 8 + g;
        // rows past row_count are never written: they take the tile's smallest limit and need no masking of their own
        limit[nt] = r < item.row_count ? ses.seq_len - (ses.q_rows - 1 - (item.row_begin + r) / group) : limit_min;
    }
    // A fragment of V^T: matrix j = lane / 8 covers keys 8 (j >> 1) .. +7, dims 8 (j & 1) .. +7 (read transposed)
    const uint32_t v_off = ((lane & 7) + (lane >> 4) * 8) * S::kRowBytes + ((lane >> 3) & 1) * 16 + head * HD * 2;

    for (uint32_t i = 0; i < n_blocks; ++i) {
        if (!warp_all(mbar_wait(&s_full[i & 1], (i >> 1) & 1))) { timed_out = true; break; }
        const float *sb = score + (i & 1) * S::kScoreTile;
        float sv[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float2 lo = *reinterpret_cast<const float2 *>(sb + (nt * 8 + g) * S::kScorePitch + 2 * t);
            const float2 hi = *reinterpret_cast<const float2 *>(sb + (nt * 8 + g) * S::kScorePitch + 2 * t + 8);
            sv[nt][0] = lo.x; sv[nt][1] = lo.y; sv[nt][2] = hi.x; sv[nt][3] = hi.y;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[i & 1]);

        // ---- mask + online softmax of row 8 nt + g over this lane's four keys ----
        const uint32_t blk_key0 = item.key_begin + i * kKeysPerBlock;
        bool plain = blk_key0 + kKeysPerBlock <= item.key_end;
        if constexpr (SINK)
            plain = plain && ses.q_rows == 1;        // one row: the union of the windows is its window
        else
            plain = plain && blk_key0 + kKeysPerBlock <= limit_min && (FORM != kPassPlain || ses.keep == nullptr);
        uint32_t pb[NT][2];
        float alpha[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float s = sv[nt][j] * scale_log2;
                if (!plain) {
                    const uint32_t key = blk_key0 + 2 * t + (j >> 1) * 8 + (j & 1);
                    bool ok = key < item.key_end;
                    if constexpr (SINK) {
                        const uint32_t at = key < extra.sink ? key : ses.kv_start + (key - extra.sink);
                        ok = ok && at < limit[nt] && (at < extra.sink || at + extra.window >= limit[nt]);
                    } else {
                        ok = ok && key < limit[nt];
                        if constexpr (FORM == kPassPlain)
                            if (ok && ses.keep != nullptr) ok = ses.keep[key] != 0;
                    }
                    s = ok ? s : -INFINITY;
                }
                sv[nt][j] = s;
                mx = fmaxf(mx, s);
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float m_new = fmaxf(m_run[nt], mx);
            const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
            alpha[nt] = fast_exp2(m_run[nt] - m_use);
            m_run[nt] = m_new;
            float pe[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pe[j] = fast_exp2(sv[nt][j] - m_use);
            pb[nt][0] = pack2<T>(pe[0], pe[1]);
            pb[nt][1] = pack2<T>(pe[2], pe[3]);
            if constexpr (FORM == kPassScores) l_true[nt] = l_true[nt] * alpha[nt] + ((pe[0] + pe[1]) + (pe[2] + pe[3]));
            // row sums from the ROUNDED weights the MMA consumes: O / l stays a convex combination
            l_run[nt] = l_run[nt] * alpha[nt] + sum2<T>(pb[nt][0]) + sum2<T>(pb[nt][1]);
        }
        // the accumulators hold query rows 2t, 2t+1: their factors live in the lanes of quad rows 2t and 2t+1
        bool rescale = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) rescale |= alpha[nt] != 1.f;
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float a0 = __shfl_sync(0xffffffffu, alpha[nt], 8 * t), a1 = __shfl_sync(0xffffffffu, alpha[nt], 8 * t + 4);
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) {
                    acc[nt][mt][0] *= a0; acc[nt][mt][1] *= a1;
                    acc[nt][mt][2] *= a0; acc[nt][mt][3] *= a1;
                }
            }
        }

        // ---- O^T += V^T P^T ----
        if (!warp_all(mbar_wait(&v_full[i % kStages], (i / kStages) & 1))) { timed_out = true; break; }
        const uint32_t stage = smem_u32(v_ring + (i % kStages) * S::kTileBytes);
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
            uint32_t a[4];
            ldmatrix_x4_trans(a, stage + v_off + mt * 32);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<T>(acc[nt][mt], a, pb[nt][0], pb[nt][1]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_empty[i % kStages]);
        if (head == 0) {
            consumed = i + 1;
            if (issued < n_blocks) {
                if (!warp_all(mbar_wait(&v_empty[i % kStages], (i / kStages) & 1))) { timed_out = true; break; }
                issue(issued, v_ring, vbase, v_full, true);
                ++issued;
            }
        }
    }

    if (timed_out) {
        for (uint32_t b = consumed; b < issued; ++b) mbar_wait(&v_full[b % kStages], (b / kStages) & 1, 1u << 16);
        if (lane == 0) atomicOr(status, TT_DEV_WAIT_TIMEOUT);
    }

    if constexpr (FORM == kPassSinkCluster) {
        // ---- (m, l, O) of this part in shared memory, then the cluster's parts of this CTA's columns ----
        constexpr uint32_t kRows = 8 * NT, kPitch = HD + 4;                    // floats per row
        static_assert((HPC * kRows * (kPitch + 2)) * 4 <= S::kRingBytes, "the parts must fit the rings");
        float *mine_o = reinterpret_cast<float *>(smem), *mine_m = mine_o + HPC * kRows * kPitch, *mine_l = mine_m + HPC * kRows;
        asm volatile("bar.sync 1, %0;" ::"n"(32 * HPC) : "memory");            // no P.V warp, hence no K.Q^T warp, reads the rings any more
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float l = l_run[nt];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (t == 0) { mine_m[head * kRows + nt * 8 + g] = m_run[nt]; mine_l[head * kRows + nt * 8 + g] = l; }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float *dst = mine_o + (head * kRows + nt * 8 + 2 * t + h) * kPitch + g;
#pragma unroll
                for (int mt = 0; mt < KS; ++mt) { dst[mt * 16] = acc[nt][mt][h]; dst[mt * 16 + 8] = acc[nt][mt][2 + h]; }
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        uint32_t rank;
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        const uint32_t vecs = HD / 4 / extra.cluster, tasks = HPC * item.row_count * vecs;
        const uint32_t o_addr = smem_u32(mine_o), m_addr = smem_u32(mine_m), l_addr = smem_u32(mine_l);
        for (uint32_t task = threadIdx.x - 32 * HPC; task < tasks; task += 32 * HPC) {
            const uint32_t row = task / vecs, col = (rank * vecs + task % vecs) * 4;
            const uint32_t hh = row / item.row_count, r = row % item.row_count, at = hh * kRows + r;
            float m[kMaxSinkCluster], l[kMaxSinkCluster];
            float4 o[kMaxSinkCluster];
#pragma unroll
            for (uint32_t i = 0; i < kMaxSinkCluster; ++i) {
                m[i] = -INFINITY; l[i] = 0.f; o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i >= extra.cluster) continue;
                uint32_t a;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(m_addr + at * 4), "r"(i));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m[i]) : "r"(a) : "memory");
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(l_addr + at * 4), "r"(i));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(l[i]) : "r"(a) : "memory");
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(o_addr + (at * kPitch + col) * 4), "r"(i));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o[i].x), "=f"(o[i].y), "=f"(o[i].z), "=f"(o[i].w) : "r"(a) : "memory");
            }
            float mx = -INFINITY;
#pragma unroll
            for (uint32_t i = 0; i < kMaxSinkCluster; ++i) mx = fmaxf(mx, m[i]);
            const float m_use = mx == -INFINITY ? 0.f : mx;                    // a row that sees nothing: all weights 0
            float d = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t i = 0; i < kMaxSinkCluster; ++i) {
                const float w = fast_exp2(m[i] - m_use);
                d = fmaf(l[i], w, d);
                sum.x = fmaf(o[i].x, w, sum.x); sum.y = fmaf(o[i].y, w, sum.y);
                sum.z = fmaf(o[i].z, w, sum.z); sum.w = fmaf(o[i].w, w, sum.w);
            }
            const float inv = d > 0.f ? 1.f / d : 0.f;
            const uint32_t packed = item.row_begin + r;
            T *dst = reinterpret_cast<T *>(ses.out) + (size_t)(packed / group) * extra.out_row_stride +
                     (size_t)((item.kv_head + hh) * group + packed % group) * HD + col;
            *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(sum.x * inv, sum.y * inv), pack2<T>(sum.z * inv, sum.w * inv));
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");      // this CTA's part has been read
        return;
    }

    // ---- write the partial: (m, l) of row 8 nt + g by the quad's first lane, O^T by everyone ----
    const uint32_t rows_total = ses.q_rows * n_q_heads;
    auto partial_row = [&](uint32_t r) {
        const uint32_t packed = item.row_begin + r;
        const uint32_t rho = (packed / group) * n_q_heads + kv_head * group + packed % group;
        return (size_t)ses.partial_base + (size_t)item.part_index * rows_total + rho;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float l = l_run[nt];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if constexpr (FORM == kPassScores) {
            l_true[nt] += __shfl_xor_sync(0xffffffffu, l_true[nt], 1);
            l_true[nt] += __shfl_xor_sync(0xffffffffu, l_true[nt], 2);
        }
        const uint32_t r = nt * 8 + g;
        if (t == 0 && r < item.row_count) {
            const size_t prow = partial_row(r);
            part_m[prow] = m_run[nt] * kLn2;   // natural-log domain, the reference's partial format
            part_l[prow] = l;
            if constexpr (FORM == kPassScores) {
                extra.part_m2[prow] = m_run[nt];
                extra.part_l2[prow] = l_true[nt];
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t ro = nt * 8 + 2 * t + h;
            if (ro >= item.row_count) continue;
            float *dst = part_o + partial_row(ro) * HD + g;
#pragma unroll
            for (int mt = 0; mt < KS; ++mt) {
                dst[mt * 16] = acc[nt][mt][h];
                dst[mt * 16 + 8] = acc[nt][mt][2 + h];
            }
        }
    }
}


template <int HD, int NT, int HPC, typename T, int FORM>
cudaError_t launch_partial_nt(cudaStream_t stream, uint32_t n_items, const TTDecodeItem *items,
                              const TTDecodeSession *sessions, float *part_o, float *part_m,
                              float *part_l, const tt_attn_batch_params *p, uint32_t *status,
                              const TTSessionTable &table, uint32_t table_keys, const PassExtra<FORM> &extra) {
    auto kernel = attn_decode_partial_kernel<HD, NT, HPC, T, FORM>;
    const int smem = DecodeSmem<HD, HPC>::kTotal;
    cudaError_t e = tt_set_smem_once(kernel, smem);
    if (e != cudaSuccess) return e;
    if constexpr (FORM == kPassSinkCluster) {
        if (extra.cluster > 8) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(n_items); cfg.blockDim = dim3(64 * HPC); cfg.dynamicSmemBytes = (size_t)smem; cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = extra.cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = tt_pdl_enabled() ? 2 : 1;
        if (extra.resident != nullptr) return cudaOccupancyMaxActiveClusters(extra.resident, kernel, &cfg);
        return cudaLaunchKernelEx(&cfg, kernel, items, sessions, part_o, part_m, part_l, p->n_q_heads, p->n_kv_heads,
                                  p->kv_token_stride_elements * 2u, p->q_row_stride_elements, p->scale * kLog2e, status, table, table_keys, extra);
    }
    return tt_launch_pdl(kernel, dim3(n_items), dim3(64 * HPC), (size_t)smem, stream, items, sessions, part_o, part_m, part_l,
                         p->n_q_heads, p->n_kv_heads, p->kv_token_stride_elements * 2u, p->q_row_stride_elements,
                         p->scale * kLog2e, status, table, table_keys, extra);
}

// `wide_rows`: some session has more than 8 packed query rows per KV head (two n-tiles per item);
// `hpc`: KV heads served by one CTA (tt_decode_heads_per_cta)
template <int HD, typename T, int FORM>
cudaError_t launch_partial(cudaStream_t stream, uint32_t n_items, const TTDecodeItem *items,
                           const TTDecodeSession *sessions, float *part_o, float *part_m,
                           float *part_l, const tt_attn_batch_params *p, uint32_t *status,
                           const TTSessionTable &table, uint32_t table_keys, bool wide_rows, uint32_t hpc,
                           const PassExtra<FORM> &extra) {
#define TT_P(NT, HPC) launch_partial_nt<HD, NT, HPC, T, FORM>(stream, n_items, items, sessions, part_o, part_m, part_l, p, status, table, table_keys, extra)
    if (hpc == 2) return wide_rows ? TT_P(2, 2) : TT_P(1, 2);
    return wide_rows ? TT_P(2, 1) : TT_P(1, 1);
#undef TT_P
}

template <typename T, int FORM>
cudaError_t launch_partial_hd(cudaStream_t stream, uint32_t n_items, const TTDecodeItem *items,
                              const TTDecodeSession *sessions, float *part_o, float *part_m,
                              float *part_l, const tt_attn_batch_params *p, uint32_t *status,
                              const TTSessionTable &table, uint32_t table_keys, bool wide_rows, uint32_t hpc,
                              const PassExtra<FORM> &extra) {
    switch (p->head_dim) {
        case 64: return launch_partial<64, T, FORM>(stream, n_items, items, sessions, part_o, part_m, part_l, p, status, table, table_keys, wide_rows, hpc, extra);
        case 128: return launch_partial<128, T, FORM>(stream, n_items, items, sessions, part_o, part_m, part_l, p, status, table, table_keys, wide_rows, hpc, extra);
        case 256: return launch_partial<256, T, FORM>(stream, n_items, items, sessions, part_o, part_m, part_l, p, status, table, table_keys, wide_rows, hpc, extra);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace
