// Eviction from a KV cache by accumulated attention weight: choose the rows to keep per KV head, compact them.
//
// Every (session, KV head) has its own statistic A[row] (tt_attn_decode_accumulate) and keeps `budget` of its `rows`
// rows: the protected ones (token position below `sink_tokens`, or among the last `recent_tokens`), then by A
// descending, ties to the lower row. Attention over a cache whose keys carry their rotation already does not depend
// on the order of its rows, so nothing is shifted: a kept row below `budget` stays where it is, and the rows given up
// there ("holes") are filled, in ascending order, by the kept rows above it. At most min(budget, rows - budget) rows
// move, one when a full cache takes in one token; sources lie at or above `budget` and destinations below it, so the
// moves are free of order and the same in place and into other buffers.
//
// kv_evict_select_kernel: one CTA or thread-block cluster per (session, KV head). The selection key of a row is 32 bits whose
//   unsigned order is the order above; a CTA keeps its slice of keys in shared memory, so the statistic and the
//   positions are read once, 16 bytes a thread where they are aligned. The budget-th largest key is found by three
//   histogram rounds (11 + 11 + 10 bits, counts of the cluster's CTAs added through distributed shared memory; a warp
//   whose keys all fall into one bin -- protected rows, rows that nothing has looked at -- adds once), then one pass gives
//   ties their rank in row order and one numbers holes and fills. A thread owns consecutive rows, an odd number of them,
//   so that ranks need one block scan and the strided shared-memory reads meet no bank twice. Bound: the latency of about
//   a dozen block or cluster barriers. Clocks for 4200 rows (one CTA of 512 threads) and 131071 (16 of 1024): loads 3700 and
//   4200, the bits of the threshold 6500 and 30,000, ties 1400 and 4700, holes and fills 4000 and 11,000; a call 13 and 34 us.
// kv_evict_move_kernel: a warp per 8 to 32 destination rows copies what changes, 16 bytes a lane; bound by HBM and, at 17 MB (10 us),
//   by its start. A session that gives up a handful of rows in place (one per step at the budget) is compacted by the selecting CTA itself: one launch.
#include "tt_sm100.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr uint32_t kMaxSelWarps = 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMaxCluster = 16;               // above 8: the non-portable size, allowed for this kernel
constexpr uint32_t kFusedMoves = 1024;             // most rows a selecting CTA moves itself
constexpr uint32_t kSelSliceKeys = 50000;          // keys a CTA holds: 200,000 bytes beside the histogram and the counters
constexpr uint32_t kRanked = 256;                  // keys that are compared with one another
constexpr uint32_t kHoleFlag = 0x80000000u;

struct EvictSession {
    const unsigned char *k, *v;
    unsigned char *k_out, *v_out;
    const float *weights;
    float *weights_out;
    const uint32_t *positions;
    uint32_t *positions_out;
    uint32_t rows;
    uint32_t end_position;
    uint32_t map_begin;          // first entry of KV head 0's map; a head's map and fill list take `map_pitch` entries
    uint32_t map_pitch;
};

struct EvictTable {
    EvictSession s[kParamSessions];
    uint32_t n;
};

struct EvictParams {
    uint32_t budget, sink, recent, n_kv_heads;
    uint32_t weight_stride, weight_out_stride;      // elements between the heads of a session
    uint32_t row_bytes;                             // one head of one row
    uint32_t held_keys;                             // selection keys a CTA's shared memory has room for
    size_t in_stride, out_stride;                   // bytes between token rows
};

// Unsigned order = order of preference. Protected rows above every weight; NaN below every weight.
__device__ __forceinline__ uint32_t evict_key(float w, bool is_protected) {
    if (is_protected) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);          // -0 counts as 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Exclusive block scan of one value per thread; *total gets the sum. Two barriers.
template <uint32_t WARPS>
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t *warp_sums, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += up;
    }
    __syncthreads();                                       // the previous use of warp_sums is over
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < WARPS; ++w) {
        const uint32_t s = warp_sums[w];
        before += w < warp ? s : 0u;
        all += s;
    }
    *total = all;
    return before + inc - x;
}

struct __align__(16) SelShared {
    uint32_t hist[kBins];
    uint32_t sum[2][kBins / 2];  // [round parity]: counts of this CTA's share of the bins over the cluster (read by the cluster)
    uint32_t warp_sums[kMaxSelWarps];
    uint32_t total[2];           // ... and their total
    uint32_t counts[4];          // this CTA's ties, holes, fills (read by the cluster)
    uint32_t before[4];          // ... of the CTAs before this one
    uint32_t owner[2];           // the CTA whose bins hold the wanted rank, keys above its bins
    uint32_t pick[3];            // the bin that holds it, keys above it, keys in it
    uint32_t hole_rows[kFusedMoves], fill_rows[kFusedMoves];
};

// CLUSTER: several CTAs per (session, head). FUSED (one CTA, in place, at most kFusedMoves rows given up): the moves too.
// 512 threads alone (a few thousand rows: barriers dominate), 1024 in a cluster.
template <bool CLUSTER, bool FUSED>
__global__ void __launch_bounds__(CLUSTER ? 1024 : 512)
kv_evict_select_kernel(const __grid_constant__ EvictTable table, EvictParams p, uint32_t *__restrict__ maps) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ SelShared sh;
    constexpr uint32_t kSelThreads = CLUSTER ? 1024 : 512, kSelWarps = kSelThreads / 32;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t size = CLUSTER ? cluster.num_blocks() : 1u, rank = CLUSTER ? cluster.block_rank() : 0u;
    auto sync_all = [&]() { if constexpr (CLUSTER) cluster.sync(); else __syncthreads(); };
    const uint32_t pair = blockIdx.x / size;
    const EvictSession ses = table.s[pair / p.n_kv_heads];
    const uint32_t head = pair % p.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    const float *weights = ses.weights + (size_t)head * p.weight_stride;
    const uint32_t *positions = ses.positions ? ses.positions + (size_t)head * p.weight_stride : nullptr;
    if (ses.rows <= p.budget) {                            // nothing is given up (the whole cluster leaves)
        if constexpr (FUSED) {
            for (uint32_t j = threadIdx.x; j < ses.rows; j += kSelThreads) {
                const size_t to = (size_t)head * p.weight_out_stride + j;
                if (ses.weights_out != ses.weights) ses.weights_out[to] = weights[j];
                if (ses.positions_out != nullptr && ses.positions_out != ses.positions) ses.positions_out[to] = positions ? positions[j] : j;
            }
        }
        return;
    }

    uint32_t *map = maps + ses.map_begin + (size_t)head * ses.map_pitch;
    uint32_t *fills = map + p.budget;
    const uint32_t slice = ((ses.rows + size - 1) / size + 3) / 4 * 4;
    const uint32_t begin = min(ses.rows, rank * slice), n = min(ses.rows, begin + slice) - begin;
    const bool held = slice <= p.held_keys;                // else every round reads the statistic again
    auto key_from = [&](float w, uint32_t pos) {
        return evict_key(w, pos < p.sink || (uint64_t)pos + p.recent >= ses.end_position);
    };
    auto key_at = [&](uint32_t i) { return key_from(weights[begin + i], positions ? positions[begin + i] : begin + i); };
    if (held) {
        // 16 bytes a thread behind the first aligned row, where the statistic and the positions share their alignment
        uint32_t head_rows = 0, quads = 0;
        if (((uintptr_t)weights ^ (positions ? (uintptr_t)positions : (uintptr_t)weights)) % 16 == 0) {
            head_rows = min(n, (uint32_t)((16 - (uintptr_t)(weights + begin) % 16) % 16 / 4));
            quads = (n - head_rows) / 4;
        }
        const float *w0 = weights + begin + head_rows;
        const uint32_t *p0 = positions + begin + head_rows;
#pragma unroll 4
        for (uint32_t c = threadIdx.x; c < quads; c += kSelThreads) {
            const float4 w = *reinterpret_cast<const float4 *>(w0 + 4 * c);
            const uint32_t i = head_rows + 4 * c;
            uint4 q = make_uint4(begin + i, begin + i + 1, begin + i + 2, begin + i + 3);
            if (positions) q = *reinterpret_cast<const uint4 *>(p0 + 4 * c);
            keys[i] = key_from(w.x, q.x); keys[i + 1] = key_from(w.y, q.y); keys[i + 2] = key_from(w.z, q.z); keys[i + 3] = key_from(w.w, q.w);
        }
        for (uint32_t i = threadIdx.x; i < head_rows; i += kSelThreads) keys[i] = key_at(i);
#pragma unroll 4
        for (uint32_t i = head_rows + quads * 4 + threadIdx.x; i < n; i += kSelThreads) keys[i] = key_at(i);
    }
    auto key_of = [&](uint32_t i) { return held ? keys[i] : key_at(i); };

    // ---- the budget-th largest key: three rounds over its bits from the top ----
    uint32_t prefix = 0, want = p.budget;                  // key bits fixed so far; rank wanted among the keys that share them
    const uint32_t share = CLUSTER ? kBins / size : kBins;      // bins whose counts a CTA adds up
    // One CTA alone: where few keys share the bits of the first round they are compared with one another instead of counted
    // twice more (4096 rows: 13.1 us to 11.7).
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
        const uint32_t bits = round < 2 ? 11u : 10u, shift = round == 0 ? 21u : round == 1 ? 10u : 0u;
        uint32_t *sum = sh.sum[round & 1];
        for (uint32_t b = threadIdx.x; b < kBins; b += kSelThreads) sh.hist[b] = 0;
        if constexpr (CLUSTER)
            if (threadIdx.x < share) sum[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll 4
        for (uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {
            const uint32_t i = i0 + threadIdx.x;
            const uint32_t key = i < n ? key_of(i) : 0u;
            const bool counts = i < n && (round == 0 || key >> (shift + bits) == prefix);
            const uint32_t counted = __ballot_sync(0xffffffffu, counts);
            if (counted == 0) continue;                    // after the first round: nearly always
            // a warp of one bin adds once; else every lane adds its own
            const uint32_t bin = (key >> shift) & ((1u << bits) - 1);
            const int first = __ffs(counted) - 1;
            const uint32_t same = __shfl_sync(0xffffffffu, bin, first);
            if (__all_sync(0xffffffffu, !counts || bin == same)) {
                if ((threadIdx.x & 31) == (uint32_t)first) atomicAdd(&sh.hist[bin], (uint32_t)__popc(counted));
            } else if (counts) {
                atomicAdd(&sh.hist[bin], 1u);
            }
        }
        sync_all();
        const uint32_t *bins = sh.hist;
        uint32_t first_bin = 0, above0 = 0;
        if constexpr (CLUSTER) {
            // every CTA adds up its share of the bins, then the share that holds the wanted rank is found from the shares'
            // totals, and its bins are read from its owner (adding up all bins in every CTA took 15,000 clocks a round)
            const uint32_t b = threadIdx.x & (share - 1), q = threadIdx.x / share, step = kSelThreads / share;
            uint32_t v = 0;
#pragma unroll 4
            for (uint32_t r = q; r < size; r += step) v += cluster.map_shared_rank(sh.hist, r)[rank * share + b];
            if (v) atomicAdd(&sum[b], v);
            __syncthreads();
            if (threadIdx.x < 32) {
                uint32_t all = 0;
                for (uint32_t x = threadIdx.x; x < share; x += 32) all += sum[x];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
                if (threadIdx.x == 0) sh.total[round & 1] = all;
            }
            cluster.sync();
            if (threadIdx.x < 32) {
                const uint32_t lane = threadIdx.x;                                   // lane i: the i-th share from the top
                const uint32_t x = lane < size ? cluster.map_shared_rank(sh.total, size - 1 - lane)[round & 1] : 0u;
                uint32_t inc = x;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= (uint32_t)o) inc += up;
                }
                if (lane < size && inc - x < want && want <= inc) { sh.owner[0] = size - 1 - lane; sh.owner[1] = inc - x; }
            }
            __syncthreads();
            bins = cluster.map_shared_rank(sum, sh.owner[0]);
            first_bin = sh.owner[0] * share;
            above0 = sh.owner[1];
        }
        // thread t takes bins kPer t .. counted from the top
        constexpr uint32_t kPer = CLUSTER ? 2 : kBins / kSelThreads;
        uint32_t c[kPer], mine = 0;
#pragma unroll
        for (uint32_t x = 0; x < kPer; ++x) c[x] = 0;
        if (kPer * threadIdx.x < share) {
            const uint32_t *from = bins + (share - kPer - kPer * threadIdx.x);
            if constexpr (kPer == 4) {
                const uint4 h = *reinterpret_cast<const uint4 *>(from);
                c[0] = h.w; c[1] = h.z; c[2] = h.y; c[3] = h.x;
            } else {
                const uint2 h = *reinterpret_cast<const uint2 *>(from);
                c[0] = h.y; c[1] = h.x;
            }
#pragma unroll
            for (uint32_t x = 0; x < kPer; ++x) mine += c[x];
        }
        uint32_t total;
        const uint32_t above = above0 + block_scan<kSelWarps>(mine, sh.warp_sums, &total);
        if (above < want && want <= above + mine) {
            uint32_t seen = above, nth = 0, in_bin = c[0];
#pragma unroll
            for (uint32_t x = 1; x < kPer; ++x)
                if (seen + in_bin < want) { seen += in_bin; in_bin = c[x]; nth = x; }
            sh.pick[0] = first_bin + share - 1 - kPer * threadIdx.x - nth;
            sh.pick[1] = seen;
            sh.pick[2] = in_bin;
        }
        if constexpr (!CLUSTER)
            if (threadIdx.x == 0) sh.owner[0] = 0;
        __syncthreads();
        prefix = (prefix << bits) | sh.pick[0];
        want -= sh.pick[1];
        if constexpr (!CLUSTER) {
            const uint32_t left = sh.pick[2];
            uint32_t *some = sh.sum[0];                    // which only clusters use
            if (round == 0 && left <= kRanked) {
                for (uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {
                    const uint32_t i = i0 + threadIdx.x;
                    const uint32_t key = i < n ? key_of(i) : 0u;
                    const bool is = i < n && key >> shift == prefix;
                    const uint32_t found = __ballot_sync(0xffffffffu, is);
                    if (found == 0) continue;
                    uint32_t at = 0;
                    if ((threadIdx.x & 31) == 0) at = atomicAdd(&sh.owner[0], (uint32_t)__popc(found));
                    at = __shfl_sync(0xffffffffu, at, 0) + __popc(found & ((1u << (threadIdx.x & 31)) - 1));
                    if (is) some[at] = key;
                }
                if (threadIdx.x >= left && threadIdx.x < (left + 3) / 4 * 4) some[threadIdx.x] = 0;          // above no key
                __syncthreads();
                if (threadIdx.x < left) {
                    const uint32_t mine = some[threadIdx.x];
                    uint32_t above = 0, same = 0;
                    for (uint32_t j = 0; j < left; j += 4) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(some + j);
                        above += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
                        same += (x.x == mine) + (x.y == mine) + (x.z == mine) + (x.w == mine);
                    }
                    if (above < want && want <= above + same) { sh.pick[0] = mine; sh.pick[1] = above; }          // one key does
                }
                __syncthreads();
                prefix = sh.pick[0];
                want -= sh.pick[1];
                __syncthreads();
                break;
            }
        }
        __syncthreads();
    }
    const uint32_t threshold = prefix, ties_kept = want;   // keys above it stay, and the first `ties_kept` equal to it

    // ---- consecutive rows per thread: rank of ties, then of holes and fills, in row order ----
    const uint32_t per = ((n + kSelThreads - 1) / kSelThreads) | 1u;
    const uint32_t i0 = min(n, threadIdx.x * per), i1 = min(n, i0 + per);
    uint32_t ties = 0;
    for (uint32_t i = i0; i < i1; ++i) ties += key_of(i) == threshold;
    uint32_t total;
    uint32_t tie_rank = block_scan<kSelWarps>(ties, sh.warp_sums, &total);
    // what the CTAs before this one have of counts[k], one read each
    auto before = [&](int k) {
        if (threadIdx.x < 32) {
            uint32_t x = 0;
            if constexpr (CLUSTER)
                if (threadIdx.x < rank) x = cluster.map_shared_rank(sh.counts, threadIdx.x)[k];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            if (threadIdx.x == 0) sh.before[k] = x;
        }
    };
    if constexpr (CLUSTER) {
        if (threadIdx.x == 0) sh.counts[0] = total;
        cluster.sync();
        before(0);
        __syncthreads();
        tie_rank += sh.before[0];
    }

    uint32_t holes = 0, kept_above = 0, t = tie_rank;
    for (uint32_t i = i0; i < i1; ++i) {
        const uint32_t key = key_of(i);
        const bool keep = key > threshold || (key == threshold && t < ties_kept);
        t += key == threshold;
        if (begin + i < p.budget) holes += !keep; else kept_above += keep;
    }
    uint32_t total_holes, total_fills;
    uint32_t hole = block_scan<kSelWarps>(holes, sh.warp_sums, &total_holes);
    uint32_t fill = block_scan<kSelWarps>(kept_above, sh.warp_sums, &total_fills);
    if constexpr (CLUSTER) {
        if (threadIdx.x == 0) { sh.counts[1] = total_holes; sh.counts[2] = total_fills; }
        cluster.sync();
        before(1);
        before(2);
        __syncthreads();
        hole += sh.before[1];
        fill += sh.before[2];
    }
    t = tie_rank;
    for (uint32_t i = i0; i < i1; ++i) {
        const uint32_t key = key_of(i), row = begin + i;
        const bool keep = key > threshold || (key == threshold && t < ties_kept);
        t += key == threshold;
        if constexpr (FUSED) {
            if (row < p.budget) {
                if (!keep) sh.hole_rows[hole++] = row;
            } else if (keep) {
                sh.fill_rows[fill++] = row;
            }
        } else {
            if (row < p.budget) {
                const uint32_t entry = keep ? row : kHoleFlag | hole++;
                if (held) keys[i] = entry; else map[row] = entry;      // a thread's rows lie apart: through shared memory
            } else if (keep) {
                fills[fill++] = row;
            }
        }
    }
    if (!FUSED && held) {
        __syncthreads();
        const uint32_t below = begin < p.budget ? min(n, p.budget - begin) : 0u;
        for (uint32_t i = threadIdx.x; i < below; i += kSelThreads) map[begin + i] = keys[i];
    }
    if constexpr (CLUSTER) cluster.sync();                 // a CTA's counters outlive their readers
    if constexpr (FUSED) {
        __syncthreads();
        const size_t out0 = (size_t)head * p.weight_out_stride;
        // statistics of other buffers: the rows that stay (holes get theirs below, in order behind a barrier)
        if (ses.weights_out != ses.weights || (ses.positions_out != nullptr && ses.positions_out != ses.positions)) {
            for (uint32_t j = threadIdx.x; j < p.budget; j += kSelThreads) {
                if (ses.weights_out != ses.weights) ses.weights_out[out0 + j] = weights[j];
                if (ses.positions_out != nullptr && ses.positions_out != ses.positions) ses.positions_out[out0 + j] = positions ? positions[j] : j;
            }
            __syncthreads();
        }
        // the moves: a group of row_bytes / 16 lanes per row, four rows' K and V in flight
        const uint32_t lanes = p.row_bytes / 16, unit = threadIdx.x / lanes, units = kSelThreads / lanes;
        const size_t off = (size_t)head * p.row_bytes + threadIdx.x % lanes * 16;
        for (uint32_t m0 = unit; m0 < total_holes; m0 += 4 * units) {
            uint4 k[4], v[4];
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
                if (m0 + x * units < total_holes) {
                    const size_t src = (size_t)sh.fill_rows[m0 + x * units] * p.in_stride + off;
                    k[x] = *reinterpret_cast<const uint4 *>(ses.k + src);
                    v[x] = *reinterpret_cast<const uint4 *>(ses.v + src);
                }
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
                if (m0 + x * units < total_holes) {
                    const size_t dst = (size_t)sh.hole_rows[m0 + x * units] * p.out_stride + off;
                    *reinterpret_cast<uint4 *>(ses.k_out + dst) = k[x];
                    *reinterpret_cast<uint4 *>(ses.v_out + dst) = v[x];
                }
        }
        for (uint32_t m = threadIdx.x; m < total_holes; m += kSelThreads) {
            const uint32_t to = sh.hole_rows[m], from = sh.fill_rows[m];
            ses.weights_out[out0 + to] = weights[from];
            if (ses.positions_out != nullptr) ses.positions_out[out0 + to] = positions ? positions[from] : from;
        }
    }
}

// grid = (blocks of 8 * ROWS destination rows, sessions x KV heads), a warp per ROWS of them: 8 into other buffers, 32 in place,
// where few of them change, but 16 of 512 bytes (32 sessions of 4096 rows give up a quarter: head_dim 256 46.9 us with 32, 41.8
// with 16; head_dim 128 and 8 KV heads 57.6 and 64.3). Up to eight rows' loads are in flight before their stores.
template <int ROW_BYTES, int ROWS>
__global__ void __launch_bounds__(256)
kv_evict_move_kernel(const __grid_constant__ EvictTable table, EvictParams p, const uint32_t *__restrict__ maps) {
    constexpr uint32_t kLanes = ROW_BYTES / 16, kAtOnce = 32 / kLanes, kRounds = 8 / kAtOnce;
    __shared__ uint8_t lists[8][32];
    const EvictSession &ses = table.s[blockIdx.y / p.n_kv_heads];
    const uint32_t head = blockIdx.y % p.n_kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t j0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * ROWS;
    const uint32_t kept = min(ses.rows, p.budget);
    if (j0 >= kept) return;
    const uint32_t j = j0 + lane;
    const bool mine = lane < ROWS && j < kept;
    uint32_t src = j;
    bool hole = false;
    if (ses.rows > p.budget && mine) {
        const uint32_t *map = maps + ses.map_begin + (size_t)head * ses.map_pitch;
        const uint32_t e = map[j];
        hole = (e & kHoleFlag) != 0;
        if (hole) src = map[p.budget + (e & ~kHoleFlag)];
    }
    // rows to copy: the holes, and every row where the destination is another buffer
    const uint32_t live = __ballot_sync(0xffffffffu, mine), holes = __ballot_sync(0xffffffffu, hole);
    const uint32_t todo_k = ses.k_out != ses.k ? live : holes, todo_v = ses.v_out != ses.v ? live : holes, todo = todo_k | todo_v;
    uint8_t *list = lists[threadIdx.x >> 5];
    if ((todo >> lane) & 1u) list[__popc(todo & ((1u << lane) - 1))] = (uint8_t)lane;
    __syncwarp();
    const uint32_t n = __popc(todo);
    const size_t head_off = (size_t)head * ROW_BYTES + (lane % kLanes) * 16;
    for (uint32_t i0 = 0; i0 < n; i0 += 8) {
        uint4 k[kRounds], v[kRounds];
#pragma unroll
        for (uint32_t i = 0; i < kRounds; ++i) {
            const uint32_t nth = i0 + i * kAtOnce + lane / kLanes, at = list[min(nth, n - 1)];
            const size_t in = (size_t)__shfl_sync(0xffffffffu, src, at) * p.in_stride + head_off;
            if (nth < n && ((todo_k >> at) & 1u)) k[i] = *reinterpret_cast<const uint4 *>(ses.k + in);
            if (nth < n && ((todo_v >> at) & 1u)) v[i] = *reinterpret_cast<const uint4 *>(ses.v + in);
        }
#pragma unroll
        for (uint32_t i = 0; i < kRounds; ++i) {
            const uint32_t nth = i0 + i * kAtOnce + lane / kLanes, at = list[min(nth, n - 1)];
            const size_t out = (size_t)(j0 + at) * p.out_stride + head_off;
            if (nth < n && ((todo_k >> at) & 1u)) *reinterpret_cast<uint4 *>(ses.k_out + out) = k[i];
            if (nth < n && ((todo_v >> at) & 1u)) *reinterpret_cast<uint4 *>(ses.v_out + out) = v[i];
        }
    }
    if (mine) {
        const size_t at = (size_t)head * p.weight_stride + src, to = (size_t)head * p.weight_out_stride + j;
        if (hole || ses.weights_out != ses.weights) ses.weights_out[to] = ses.weights[at];
        if (ses.positions_out != nullptr && (hole || ses.positions_out != ses.positions))
            ses.positions_out[to] = ses.positions ? ses.positions[at] : src;
    }
}

// CTAs per (session, KV head). The rounds of a cluster cost three times those of a CTA alone, so up to 10000 rows stay with
// one (9000 rows of 16 sessions x 2 heads: 23 us, 32 with two); beyond, slices of some 2048 rows while half of the SMs
// have room for them (16000 rows of 4 sessions: 21.7 us, 25.5 with slices of 8192), and enough CTAs that the slices
// fit shared memory.
uint32_t cluster_size(uint32_t max_rows, uint32_t pairs, uint32_t sm_count) {
    uint32_t c = 1;
    while (c < kMaxCluster && ((max_rows > (c == 1 ? 10000u : c * 2048u) && (uint64_t)pairs * c * 4 <= sm_count) || (uint64_t)c * kSelSliceKeys < max_rows))
        c *= 2;
    return c;
}

// Rows the selecting CTA moves itself rather than a second launch: a CTA moves some 73 GB/s, so it pays with few rows or many
// CTAs (4096 rows of 512 bytes a head, 410 given up: 2 CTAs 17.1 us against 13.7, 32 17.2 against 20.6, 128 24.4 against 53.5;
// 614 given up: 32 CTAs 21.9 both ways, 64 25.3 against 39.1; 1024: 33.9 against 42.4).
uint32_t fused_moves(uint32_t pairs) { return pairs >= 64 ? kFusedMoves : pairs >= 32 ? kFusedMoves / 2 : kFusedMoves / 4; }

// entries of a head's map: a source for every kept row, and the list of the rows that fill holes
uint64_t map_entries(uint32_t rows, uint32_t budget) {
    return rows <= budget ? 0 : (uint64_t)budget + (rows - budget < budget ? rows - budget : budget);
}

bool overlaps(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + b_bytes && y < x + a_bytes;
}

template <bool CLUSTER, bool FUSED>
cudaError_t launch_select(cudaStream_t stream, const EvictTable &table, const EvictParams &p, uint32_t ctas, uint32_t cluster, uint32_t *maps) {
    auto kernel = kv_evict_select_kernel<CLUSTER, FUSED>;
    cudaError_t e = tt_set_smem_once(kernel, (int)(kSelSliceKeys * sizeof(uint32_t)));
    if (e != cudaSuccess) return e;
    if (CLUSTER && cluster > 8) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(CLUSTER ? 1024 : 512); cfg.dynamicSmemBytes = sizeof(uint32_t) * p.held_keys; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = tt_pdl_enabled() ? attr : attr + 1;
    cfg.numAttrs = (tt_pdl_enabled() ? 1 : 0) + (CLUSTER ? 1 : 0);
    return cudaLaunchKernelEx(&cfg, kernel, table, p, maps);
}

// `given_up`: most rows a session gives up; `in_place`: K and V of every session
cudaError_t launch_evict(tt_context *ctx, cudaStream_t stream, const EvictTable &table, EvictParams p, uint32_t max_rows,
                         uint32_t given_up, bool in_place, uint32_t *maps) {
    const uint32_t pairs = table.n * p.n_kv_heads;
    cudaError_t e = cudaSuccess;
    if (given_up != 0) {
        const uint32_t c = cluster_size(max_rows, pairs, (uint32_t)ctx->sm_count);
        const uint32_t slice = ((max_rows + c - 1) / c + 3) / 4 * 4;
        p.held_keys = slice <= kSelSliceKeys ? slice : kSelSliceKeys;
        const bool fused = c == 1 && in_place && given_up <= fused_moves(pairs);
        e = fused ? launch_select<false, true>(stream, table, p, pairs, 1, maps)
                  : c == 1 ? launch_select<false, false>(stream, table, p, pairs, 1, maps)
                           : launch_select<true, false>(stream, table, p, pairs * c, c, maps);
        if (e != cudaSuccess) return e;
        ctx->launches++;
        if (fused) return cudaSuccess;
    }
    const uint32_t kept = max_rows < p.budget ? max_rows : p.budget;
    if (kept == 0) return cudaSuccess;
    const uint32_t rows = !in_place ? 8 : p.row_bytes == 512 ? 16 : 32;
    const dim3 grid((kept + 8 * rows - 1) / (8 * rows), pairs);
#define TT_X(BYTES) e = in_place ? tt_launch_pdl(kv_evict_move_kernel<BYTES, BYTES == 512 ? 16 : 32>, grid, dim3(256), 0, stream, table, p, maps) \
                                 : tt_launch_pdl(kv_evict_move_kernel<BYTES, 8>, grid, dim3(256), 0, stream, table, p, maps)
    if (p.row_bytes == 128) TT_X(128);
    else if (p.row_bytes == 256) TT_X(256);
    else TT_X(512);
#undef TT_X
    if (e == cudaSuccess) ctx->launches++;
    return e;
}

}  // namespace

TT_API int tt_kv_evict(tt_context *ctx, tt_stream stream, const tt_kv_evict_session *sessions, uint32_t n_sessions,
                       const tt_kv_evict_params *params) {
    TT_ENTER(ctx);
    if (params == nullptr || (sessions == nullptr && n_sessions != 0))
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "sessions and params must not be null");
    const tt_kv_evict_params &q = *params;
    if (q.head_dim != 64 && q.head_dim != 128 && q.head_dim != 256)
        return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "eviction supports head_dim 64/128/256, got %u", q.head_dim);
    if (q.n_kv_heads == 0 || q.n_kv_heads > 96) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_kv_heads must be in 1..96");
    if (q.budget == 0 || q.budget > (uint32_t)INT32_MAX) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "budget must be in 1..2^31-1");
    if ((uint64_t)q.sink_tokens + q.recent_tokens > q.budget)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "%u sinks and %u recent rows exceed the budget of %u rows", q.sink_tokens,
                            q.recent_tokens, q.budget);
    const uint64_t width = (uint64_t)q.n_kv_heads * q.head_dim;
    const uint64_t in_stride = q.kv_token_stride_elements ? q.kv_token_stride_elements : width;
    const uint64_t out_stride = q.kv_out_token_stride_elements ? q.kv_out_token_stride_elements : in_stride;
    const uint32_t weight_out_stride = q.weight_out_head_stride ? q.weight_out_head_stride : q.weight_head_stride;
    if (in_stride < width || out_stride < width) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "a row stride is smaller than its tight width");
    if (in_stride % 8 || out_stride % 8) return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "row strides must keep rows 16-byte aligned");
    // the maps of one launch pair live in the workspace; a batch that needs more is taken in several
    uint64_t map_room = ctx->workspace_bytes / sizeof(uint32_t);
    if (map_room > UINT32_MAX) map_room = UINT32_MAX;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        const tt_kv_evict_session &s = sessions[i];
        if (s.k == nullptr || s.v == nullptr || s.weights == nullptr)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u has a null buffer", i);
        if (((uintptr_t)s.k | (uintptr_t)s.v | (uintptr_t)s.k_out | (uintptr_t)s.v_out) & 15)
            return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "session %u: K and V must be 16-byte aligned", i);
        if (((uintptr_t)s.weights | (uintptr_t)s.weights_out | (uintptr_t)s.positions | (uintptr_t)s.positions_out) & 3)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: weights and positions must be 4-byte aligned", i);
        if (s.rows > (uint32_t)INT32_MAX || s.rows > q.weight_head_stride)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: %u rows do not fit a weight row of %u", i, s.rows, q.weight_head_stride);
        const uint32_t kept = s.rows < q.budget ? s.rows : q.budget;
        if (kept > weight_out_stride)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: %u kept rows do not fit a weight row of %u", i, kept, weight_out_stride);
        if ((s.k_out == nullptr || s.k_out == s.k || s.v_out == nullptr || s.v_out == s.v) && out_stride != in_stride)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: in place, the row strides must be equal", i);
        const bool w_in = s.weights_out == nullptr || s.weights_out == s.weights;
        const bool p_in = s.positions != nullptr && (s.positions_out == nullptr || s.positions_out == s.positions);
        if ((w_in || p_in) && weight_out_stride != q.weight_head_stride)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: in place, the weight strides must be equal", i);
        const size_t in_bytes = (size_t)s.rows * in_stride * 2, out_bytes = (size_t)kept * out_stride * 2;
        const size_t w_bytes = ((size_t)(q.n_kv_heads - 1) * q.weight_head_stride + s.rows) * 4;
        const size_t wo_bytes = ((size_t)(q.n_kv_heads - 1) * weight_out_stride + kept) * 4;
        if ((s.k_out != nullptr && s.k_out != s.k && overlaps(s.k, in_bytes, s.k_out, out_bytes)) ||
            (s.v_out != nullptr && s.v_out != s.v && overlaps(s.v, in_bytes, s.v_out, out_bytes)) ||
            (!w_in && overlaps(s.weights, w_bytes, s.weights_out, wo_bytes)) ||
            (s.positions != nullptr && !p_in && overlaps(s.positions, w_bytes, s.positions_out, wo_bytes)))
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: an output overlaps its input without being it", i);
        // before the first launch: a call refused behind it would have emptied some caches and not others
        if (map_entries(s.rows, q.budget) * q.n_kv_heads > map_room)
            return tt_set_error(ctx, TT_ERR_OOM, "the row map of session %u does not fit the context workspace", i);
    }
    EvictParams p;
    p.budget = q.budget; p.sink = q.sink_tokens; p.recent = q.recent_tokens; p.n_kv_heads = q.n_kv_heads;
    p.weight_stride = q.weight_head_stride; p.weight_out_stride = weight_out_stride;
    p.row_bytes = q.head_dim * 2; p.held_keys = 0;
    p.in_stride = in_stride * 2; p.out_stride = out_stride * 2;
    static thread_local EvictTable table;
    uint32_t i = 0;
    while (i < n_sessions) {
        uint64_t used = 0;
        uint32_t max_rows = 0, given_up = 0;
        bool in_place = true;
        table.n = 0;
        for (; i < n_sessions && table.n < kParamSessions; ++i) {
            const tt_kv_evict_session &s = sessions[i];
            const uint64_t pitch = map_entries(s.rows, q.budget);
            if (used + pitch * q.n_kv_heads > map_room) break;           // each alone fits
            EvictSession &d = table.s[table.n++];
            d.k = (const unsigned char *)s.k; d.v = (const unsigned char *)s.v;
            d.k_out = (unsigned char *)(s.k_out ? s.k_out : s.k); d.v_out = (unsigned char *)(s.v_out ? s.v_out : s.v);
            d.weights = s.weights; d.weights_out = s.weights_out ? s.weights_out : s.weights;
            d.positions = s.positions; d.positions_out = s.positions_out ? s.positions_out : s.positions;
            d.rows = s.rows; d.end_position = s.end_position;
            d.map_begin = (uint32_t)used; d.map_pitch = (uint32_t)pitch;
            used += pitch * q.n_kv_heads;
            in_place = in_place && d.k_out == d.k && d.v_out == d.v;
            if (s.rows > q.budget && s.rows - q.budget > given_up) given_up = s.rows - q.budget;
            if (s.rows > max_rows) max_rows = s.rows;
        }
        const cudaError_t e = launch_evict(ctx, (cudaStream_t)stream, table, p, max_rows, given_up, in_place, reinterpret_cast<uint32_t *>(ctx->partials));
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "kv_evict launch");
    }
    return TT_OK;
}
