// Decode attention of sessions that share a long prefix.
//
// The sessions of a group continue the same tokens (a system prompt, a document, the branches of one search), so the
// prefix's K/V rows exist once and every session's query rows see all of them. A batched decode would stream them once
// per session; here the query rows of the whole group are packed into one operand and the prefix is streamed once per
// 128 of them (64 where no group has more, 256 at head_dim 256 where one has more than 128):
//
//   prefix pass   attn_rows_kernel / attn_pair_kernel: (group, kv head, packed rows, key range) per CTA or pair on tcgen05
//                                                                                              -> (m, l, o) partials
//   suffix pass   the split-KV decode kernel over every session's own rows                            -> (m, l, o) partials
//   merge         attn_prefix_merge_kernel: log-sum-exp over both kinds of partials of an output row
//
// Where that is faster (tt_attn_decode_shared_prefix) the suffixes are items of the prefix pass and there is no suffix pass.
//
// The prefix pass (attn_rows_tc.cuh) packs row = (query row of the group) * G + g with G query heads per KV head, session
// after session. Every row of an item sees every key of its range: only the last tile of a prefix is masked. What
// bounds the pass depends on the rows: with up to about 256 packed rows per KV head the bytes of the prefix, beyond
// that the tensor pipe and the exponentials. 64 sessions of 16/2 heads behind 32768 keys (512 packed rows per KV head):
// own rows 16 us (67 MB, 4.2 TB/s), prefix pass 36 us (954 TFLOP/s), merge 7 us (24 MB of partials), a call 56 to 60 us;
// as 64 sessions of 33,000 keys each the same batch would read 4.3 GB, 660 us.
#include "attn_merge.cuh"
#include "attn_pair_tc.cuh"

#include <algorithm>

namespace {

constexpr uint32_t kParamGroups = 8;
constexpr uint32_t kFusedSessions = kParamSessions;                // sessions whose own rows may join the prefix pass
// What the parameters have room for: a launch pays for their size (25 KB against 9: 1.4 us of host time a launch, a prefix call of
// one session that is waited for 27.9 us against 25.0), so a form takes the smaller table where that is enough.
constexpr uint32_t kTableGroups = kParamGroups + kFusedSessions, kFewGroups = kParamGroups + 16;

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
    // sessions of q_rows query rows each whose queries lie q_step bytes apart (the slots of one tensor): a row's address is
    // arithmetic. q_rows 0: anything else, found by a search over the sessions -- divergent reads of the parameter bank,
    // 3000 clocks at the start of every CTA for 64 sessions.
    uint32_t q_rows;
    const void *q;
    long long q_step;
    uint32_t causal_rows;                // of a session's own rows: its query rows, of which row r sees prefix_len - (rows - 1 - r) keys
    uint32_t pad;
};
struct alignas(64) PrefixMaps { unsigned char m[2][128]; };    // K and V tensor maps of a group

// Calls of up to kParamGroups groups and kParamSessions sessions carry their tables and tensor maps in the kernel
// parameters; larger ones read the copies the host uploaded.
template <uint32_t GROUPS>
struct alignas(64) PrefixTable {
    uint32_t n_groups, n_sessions;
    uint32_t in_params;
    uint32_t item_begin[GROUPS];
    PrefixGroup g[GROUPS];
    PrefixMaps maps[GROUPS];
    PrefixSession s[kParamSessions];
};

// The prefix pass's items for attn_rows_kernel.
template <uint32_t GROUPS>
struct PrefixForm {
    static constexpr bool kPartials = true;
    // what every CTA reads first stands first and together: every line of the parameters it touches costs a miss, some 600
    // clocks each and one after the other
    uint32_t n_q_heads, n_kv_heads, q_row_stride;
    uint32_t behind_own_rows;            // the launch before this one is the pass over the sessions' own rows
    const PrefixGroup *groups;           // device copies, when !table.in_params
    const PrefixSession *sessions;
    const PrefixMaps *maps;
    float *part_o, *part_m, *part_l;
    PrefixTable<GROUPS> table;

    struct Item : RowsItem {
        const CUtensorMap *maps;
        uint32_t key_begin, n_keys;
        uint32_t causal_rows, causal_end;    // PrefixGroup.causal_rows, and the last of those rows' end behind key_begin
        uint32_t row0, n_rows;           // first packed row, packed rows in use
        uint32_t row_begin, session_begin, session_count, q_rows;
        const void *q;
        long long q_step;
        size_t partial_base;             // of packed row 0's query row in this part
    };
    __device__ __forceinline__ Item item(uint32_t block, int hd, int rows) const {
        uint32_t lo = 0, hi = table.n_groups;
        if (table.in_params) {
#pragma unroll
            for (uint32_t i = 1; i < kParamGroups; ++i)
                if (i < hi && table.item_begin[i] <= block) lo = i;
            if (hi > kParamGroups && table.item_begin[kParamGroups] <= block) {
                lo = kParamGroups;
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (table.item_begin[mid] <= block) lo = mid; else hi = mid;
                }
            }
        } else {
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (groups[mid].item_begin <= block) lo = mid; else hi = mid;
            }
        }
        const PrefixGroup grp = table.in_params ? table.g[lo] : groups[lo];
        const uint32_t local = block - grp.item_begin, group = n_q_heads / n_kv_heads;
        const uint32_t part = local / (grp.row_tiles * n_kv_heads);
        Item it;
        it.maps = reinterpret_cast<const CUtensorMap *>(table.in_params ? table.maps[lo].m[0] : maps[lo].m[0]);
        it.kv_head = local / grp.row_tiles % n_kv_heads;
        it.key_begin = min(grp.prefix_len, part * grp.part_len);
        it.n_keys = min(grp.prefix_len, it.key_begin + grp.part_len) - it.key_begin;
        it.n_tiles = (it.n_keys + kBK - 1) / kBK;
        it.n_halves = (it.n_keys + 63) / 64;
        it.causal_rows = grp.causal_rows; it.causal_end = grp.prefix_len - it.key_begin;
        it.row0 = local % grp.row_tiles * rows;
        it.n_rows = min((uint32_t)rows, grp.n_rows * group - it.row0);
        it.row_begin = grp.row_begin; it.session_begin = grp.session_begin; it.session_count = grp.session_count;
        it.q_rows = grp.q_rows; it.q = grp.q; it.q_step = grp.q_step;
        it.partial_base = (size_t)grp.partial_base + (size_t)part * grp.n_rows * n_q_heads;
        return it;
    }
    __device__ __forceinline__ const void *query(const Item &it, uint32_t r, int hd, int rows) const {
        if (r >= it.n_rows) return nullptr;
        const uint32_t group = n_q_heads / n_kv_heads, packed = it.row0 + r;
        if (it.q_rows != 0) {
            const uint32_t t = packed / group;
            return reinterpret_cast<const unsigned char *>(it.q) + (long long)(t / it.q_rows) * it.q_step +
                   ((size_t)(t % it.q_rows) * q_row_stride + (size_t)(it.kv_head * group + packed % group) * hd) * 2;
        }
        const PrefixSession *s = table.in_params ? table.s : sessions;
        const uint32_t qrow = it.row_begin + packed / group;
        uint32_t lo = it.session_begin, hi = it.session_begin + it.session_count;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (s[mid].first_row <= qrow) lo = mid; else hi = mid;
        }
        return reinterpret_cast<const unsigned char *>(s[lo].q) +
               ((size_t)(qrow - s[lo].first_row) * q_row_stride + (size_t)(it.kv_head * group + packed % group) * hd) * 2;
    }
    __device__ __forceinline__ bool waits_late() const { return behind_own_rows != 0; }
    __device__ __forceinline__ void acquire(const Item &it) const {
        if (table.in_params) return;
        // the maps were rewritten by a host copy since the last launch that used these addresses
        asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(it.maps) : "memory");
        asm volatile("fence.proxy.tensormap::generic.acquire.gpu [%0], 128;" ::"l"(it.maps + 1) : "memory");
    }
    __device__ __forceinline__ const CUtensorMap *box(const Item &it, uint32_t tile, uint32_t half, bool is_k, int &row) const {
        row = (int)(it.key_begin + tile * kBK + half * 64);
        return is_k ? it.maps : it.maps + 1;
    }
    __device__ __forceinline__ bool masked(const Item &it, uint32_t tile) const {
        return (tile + 1) * kBK > it.n_keys || (it.causal_rows > 1 && (tile + 1) * kBK + it.causal_rows - 1 > it.causal_end);
    }
    __device__ __forceinline__ void visible(const Item &it, uint32_t row, uint32_t tile, uint32_t (&bits)[4]) const {
        uint32_t end = it.n_keys;
        if (it.causal_rows > 1) {
            const uint32_t w = min((it.row0 + row) / (n_q_heads / n_kv_heads), it.causal_rows - 1), later = it.causal_rows - 1 - w;
            end = min(end, it.causal_end > later ? it.causal_end - later : 0u);
        }
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) bits[c4] = bits_between(0, (int)end - (int)(tile * kBK) - c4 * 32);
    }
    __device__ __forceinline__ bool exists(const Item &it, uint32_t r) const { return r < it.n_rows; }
    __device__ __forceinline__ size_t partial(const Item &it, uint32_t r, int rows) const {
        const uint32_t group = n_q_heads / n_kv_heads, packed = it.row0 + r;
        return it.partial_base + (size_t)(packed / group) * n_q_heads + it.kv_head * group + packed % group;
    }
};

// Draft rows over sinks and a window (tt_attn_decode_sink_window with more than the 16 packed rows of a split-KV item):
// every session is a group, and its keys are numbered in whole halves of 64: those over [0, sink), those of the windows from
// `base` on up to the ring's end, those behind it. Nothing that no row sees is multiplied: V has a map for each of the three
// ranges that ends with it. (What K has there makes scores that are replaced.)
template <uint32_t GROUPS>
struct SinkRowsForm : PrefixForm<GROUPS> {
    using Base = PrefixForm<GROUPS>;
    static constexpr uint32_t kSessions = GROUPS / 2;            // two groups' maps each
    uint32_t sink, window;
    // keys base .. base + straight - 1 are rows first_row on, the later ones rows sink on
    struct Session { uint32_t seq_len, q_rows, base, windowed, first_row, straight; } session[kSessions];

    struct Item : Base::Item {
        Session s;
        uint32_t sink_keys, straight_keys;      // key numbers that stand for the sinks, for the first range of the window
        const CUtensorMap *v_ends;              // of the sinks, of the range behind the ring's end
    };
    __device__ __forceinline__ Item item(uint32_t block, int hd, int rows) const {
        Item it;
        static_cast<typename Base::Item &>(it) = Base::item(block, hd, rows);
        it.s = session[it.session_begin];
        it.sink_keys = it.s.windowed ? (sink + 63) / 64 * 64 : 0u;
        // with nothing behind the ring's end the first range also takes the numbers past its last half: of a cache without sinks
        // they would else be row 0 of the last range's map, which cannot be empty, and a spare half of the last tile would read it
        const bool behind = it.s.seq_len - it.s.base > it.s.straight;
        it.straight_keys = behind ? (it.s.straight + 63) / 64 * 64 : 0xffffffffu;
        it.v_ends = reinterpret_cast<const CUtensorMap *>(this->table.maps[kSessions + it.session_begin].m[0]);
        return it;
    }
    __device__ __forceinline__ const CUtensorMap *box(const Item &it, uint32_t tile, uint32_t half, bool is_k, int &row) const {
        uint32_t c = it.key_begin + tile * kBK + half * 64;
        if (c < it.sink_keys) {
            row = (int)c;
            return is_k ? it.maps : it.v_ends;
        }
        c -= it.sink_keys;
        if (c < it.straight_keys) {
            row = (int)(it.s.first_row + c);
            return is_k ? it.maps : it.maps + 1;
        }
        row = (int)(sink + (c - it.straight_keys));
        return is_k ? it.maps : it.v_ends + 1;
    }
    __device__ __forceinline__ bool masked(const Item &it, uint32_t tile) const {
        uint32_t c = it.key_begin + tile * kBK;
        if (c < it.sink_keys) return true;
        c -= it.sink_keys;
        uint32_t key = it.s.base + c;
        if (c >= it.straight_keys) key = it.s.base + it.s.straight + (c - it.straight_keys);
        else if (c + kBK > it.s.straight) return true;
        return key + kBK + it.s.q_rows - 1 > it.s.seq_len || (it.s.windowed && key < max(sink, it.s.seq_len - window));
    }
    __device__ __forceinline__ void visible(const Item &it, uint32_t row, uint32_t tile, uint32_t (&bits)[4]) const {
        const uint32_t w = min((it.row0 + row) / (this->n_q_heads / this->n_kv_heads), it.s.q_rows - 1);
        const uint32_t end = it.s.seq_len - (it.s.q_rows - 1 - w);
        const uint32_t from = it.s.windowed ? max(sink, end > window ? end - window : 0u) : 0u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t c = it.key_begin + tile * kBK + half * 64, first = 0, to = end, key0 = c;
            if (c < it.sink_keys) {
                to = min(end, sink);
            } else {
                c -= it.sink_keys;
                first = from;
                if (c < it.straight_keys) {
                    key0 = it.s.base + c;
                    to = min(end, it.s.base + it.s.straight);
                } else {
                    key0 = it.s.base + it.s.straight + (c - it.straight_keys);
                }
            }
            const int lo = (int)first - (int)key0, hi = (int)to - (int)key0;
            bits[2 * half] = bits_between(lo, hi);
            bits[2 * half + 1] = bits_between(lo - 32, hi - 32);
        }
    }
};

// ---------------------------------------------------------------------------------------
// Merge (attn_merge.cuh): the row's partials of its group's prefix, then the session's own.
// ---------------------------------------------------------------------------------------
struct MergeSession {
    void *out;
    uint32_t q_rows;                     // this session's query rows
    uint32_t prefix_base, prefix_parts;  // partial rows of this session's first query row in its group's prefix pass
    uint32_t prefix_stride;              // partial rows between two parts of the prefix
    uint32_t own_base, own_parts;        // the session's own split partials
};
struct MergeTable {
    uint32_t n;                          // 0: the device copy
    uint32_t q_rows;                     // of every session; 0: they differ
    uint32_t first_row[kParamSessions];  // query rows of the call before each session
    MergeSession s[kParamSessions];
};

template <typename T, int HD>
__global__ void __launch_bounds__(256)
attn_prefix_merge_kernel(const __grid_constant__ MergeTable table, const MergeSession *__restrict__ dev,
                         const uint32_t *__restrict__ dev_first_row, uint32_t n_sessions,
                         const float *__restrict__ pre_o, const float *__restrict__ pre_m, const float *__restrict__ pre_l,
                         const float *__restrict__ own_o, const float *__restrict__ own_m, const float *__restrict__ own_l,
                         uint32_t n_q_heads, uint32_t out_row_stride, uint32_t n_rows, uint32_t groups) {
    using M = RowMerge<HD>;
    __shared__ typename M::Shared shared;
    pdl_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t out_row = M::row(blockIdx.x, warp, groups);
    const bool live = out_row < n_rows;
    const uint32_t qrow = out_row / n_q_heads, head = out_row - qrow * n_q_heads;
    uint32_t lo = 0;
    const uint32_t *first_row = table.n != 0 ? table.first_row : dev_first_row;
    if (table.q_rows != 0) {
        lo = min(qrow / table.q_rows, n_sessions - 1);
    } else {
        uint32_t hi = n_sessions;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (first_row[mid] <= qrow) lo = mid; else hi = mid;
        }
    }
    const uint32_t w = table.q_rows != 0 ? qrow - lo * table.q_rows : qrow - first_row[lo];
    const MergeSession ses = table.n != 0 ? table.s[lo] : dev[lo];

    pdl_wait();       // the partials are there
    M merge(warp, lane, groups);
    if (live) {
        merge.walk(pre_o, pre_m, pre_l, (size_t)ses.prefix_base + w * n_q_heads + head, ses.prefix_stride, ses.prefix_parts);
        merge.walk(own_o, own_m, own_l, (size_t)ses.own_base + w * n_q_heads + head, (size_t)ses.q_rows * n_q_heads, ses.own_parts);
    }
    if (!merge.join(shared) || !live) return;
    merge.template store<T>(reinterpret_cast<T *>(ses.out) + (size_t)w * out_row_stride + (size_t)head * HD);
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// Packed rows one item of the prefix pass takes: 64 when no group has more, else 128 on one SM, and 256 on a pair of SMs
// where a group has more than 128 at head_dim 256.
uint32_t rows_per_tile(const uint32_t *query_rows, uint32_t n_groups, uint32_t group, uint32_t head_dim) {
    uint64_t most = 0;
    for (uint32_t g = 0; g < n_groups; ++g) most = (uint64_t)query_rows[g] * group > most ? (uint64_t)query_rows[g] * group : most;
    return most <= 64 ? 64 : most > 128 && head_dim == 256 ? 256 : 128;
}

template <typename T, class Form>
cudaError_t launch_prefix(cudaStream_t stream, uint32_t head_dim, uint32_t rows, uint32_t n_items, const RowsParams &p, uint32_t *status,
                          const Form &form) {
#define TT_X(HD) (rows == 64 ? launch_rows<T, HD, 64>(stream, n_items, p, status, form) : launch_rows<T, HD, 128>(stream, n_items, p, status, form))
    if (rows == 256) return launch_pair<T>(stream, n_items, p, status, form);
    return head_dim == 64 ? TT_X(64) : head_dim == 128 ? TT_X(128) : TT_X(256);
#undef TT_X
}

template <typename T, class Form>
cudaError_t launch_merge(cudaStream_t stream, uint32_t head_dim, uint32_t rows, uint32_t parts, const MergeTable &table, const MergeSession *dev,
                         const uint32_t *dev_first_row, uint32_t n_sessions, const Form &kp, const TTDecodeForm &own,
                         uint32_t n_q_heads, uint32_t out_row_stride, uint32_t sm_count) {
    uint32_t grid = 0;
    const uint32_t groups = merge_groups(rows, parts, head_dim, sm_count, &grid);
#define TT_X(HD) tt_launch_pdl(attn_prefix_merge_kernel<T, HD>, dim3(grid), dim3(256), 0, stream, table, dev, dev_first_row, n_sessions, \
                               kp.part_o, kp.part_m, kp.part_l, own.part_o, own.part_m, own.part_l, n_q_heads, out_row_stride, rows, groups)
    return head_dim == 64 ? TT_X(64) : head_dim == 128 ? TT_X(128) : TT_X(256);
#undef TT_X
}

}  // namespace

// One CTA is resident per SM (an item of 256 rows takes two), and an item costs some tiles besides its own: 3 on one SM, 6
// on a pair. The length of the items is the one for which the launch takes the least time: the waves of the full-size
// items, whose last one leaves places for the short ones (short groups, a session's own rows), and what of these does not
// fit behind it. (16 sessions of 4 rows behind four prefixes of 12,000 to 16,000 keys: items of 18 tiles 41.8 us, of 15,
// whose waves are shorter but leave no room, 48.1.) Equal times go to the longer items (fewer partials to merge).
TT_API int tt_attn_plan_prefix_splits(const uint32_t *prefix_lens, const uint32_t *query_rows, uint32_t n_groups, uint32_t head_dim,
                                      uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t sm_count, size_t workspace_bytes,
                                      uint32_t *out_keys_per_item, uint32_t *out_n_items) {
    if (prefix_lens == nullptr || query_rows == nullptr || n_groups == 0 || n_kv_heads == 0 || n_q_heads == 0 ||
        n_q_heads % n_kv_heads != 0 || head_dim == 0 || sm_count == 0)
        return TT_ERR_INVALID_ARG;
    const uint32_t group = n_q_heads / n_kv_heads, tile_rows = rows_per_tile(query_rows, n_groups, group, head_dim);
    const uint64_t slots = tile_rows == 256 ? sm_count / 2 : sm_count;          // items that run at once
    const uint64_t item_tiles = tile_rows == 256 ? 6 : 3;
    if (slots == 0) return TT_ERR_INVALID_ARG;
    uint32_t longest = 0;
    for (uint32_t g = 0; g < n_groups; ++g) longest = prefix_lens[g] > longest ? prefix_lens[g] : longest;
    const uint32_t max_tiles = longest == 0 ? 1 : ceil_div(longest, kBK);
    uint64_t best = ~0ull, best_items = 0;
    uint32_t best_tiles = 0;
    for (uint32_t parts = 1; parts <= 512 && parts <= max_tiles; ++parts) {
        const uint32_t tiles = ceil_div(max_tiles, parts);
        if (parts > 1 && tiles == ceil_div(max_tiles, parts - 1)) continue;      // the same item length again
        uint64_t full = 0, longest_item = 0, few = 0, few_cost = 0, prows = 0;
        for (uint32_t g = 0; g < n_groups; ++g) {
            const uint64_t own_tiles = ceil_div(prefix_lens[g], kBK), p = ceil_div(own_tiles, tiles);
            if (p == 0) continue;
            const uint64_t n = p * n_kv_heads * ceil_div((uint64_t)query_rows[g] * group, tile_rows), each = ceil_div(own_tiles, p) + item_tiles;
            if (2 * each > tiles + item_tiles) {
                full += n;
                if (each > longest_item) longest_item = each;
            } else {
                few += n;
                few_cost += n * each;
            }
            prows += p * query_rows[g] * n_q_heads;
        }
        if (workspace_bytes != 0 && prows * ((uint64_t)head_dim + 2) * sizeof(float) > workspace_bytes) break;    // more parts need more
        const uint64_t items = full + few, waves = (full + slots - 1) / slots, mean = few != 0 ? (few_cost + few - 1) / few : 1;
        const uint64_t beside = (waves * slots - full) * (longest_item / mean), left = few > beside ? few - beside : 0;
        const uint64_t time = waves * longest_item + (left + slots - 1) / slots * mean;
        if (time < best) { best = time; best_tiles = tiles; best_items = items; }
    }
    if (best_tiles == 0) return TT_ERR_OOM;
    if (out_keys_per_item) *out_keys_per_item = best_tiles * kBK;
    if (out_n_items) *out_n_items = (uint32_t)best_items;
    return TT_OK;
}

// The launches of a call whose groups are checked; `fused`: the sessions' own rows are groups of the prefix pass too.
template <uint32_t GROUPS>
static int shared_prefix(tt_context *ctx, tt_stream stream, const tt_attn_prefix *groups, uint32_t n_groups, const tt_attn_session *sessions,
                         uint32_t n_sessions, const tt_attn_batch_params *params, bool in_params, bool fused) {
    const tt_attn_batch_params &q = *params;
    // host tables: the parameter blocks, or the staging copy of what is uploaded
    static thread_local PrefixForm<GROUPS> kp;
    PrefixTable<GROUPS> &table = kp.table;
    static thread_local MergeTable merge;
    const size_t off_groups = sizeof(PrefixMaps) * (size_t)n_groups, off_sessions = off_groups + sizeof(PrefixGroup) * (size_t)n_groups;
    const size_t off_merge = (off_sessions + sizeof(PrefixSession) * (size_t)n_sessions + 15) / 16 * 16;
    const size_t off_first = off_merge + sizeof(MergeSession) * (size_t)n_sessions;
    const size_t table_bytes = off_first + sizeof(uint32_t) * (size_t)n_sessions;
    unsigned char *host = ctx->h_prefix_tables;
    PrefixMaps *h_maps = in_params ? table.maps : reinterpret_cast<PrefixMaps *>(host);
    PrefixGroup *h_groups = in_params ? table.g : reinterpret_cast<PrefixGroup *>(host + off_groups);
    PrefixSession *h_sessions = in_params ? table.s : reinterpret_cast<PrefixSession *>(host + off_sessions);
    MergeSession *h_merge = in_params ? merge.s : reinterpret_cast<MergeSession *>(host + off_merge);
    uint32_t *h_first = in_params ? merge.first_row : reinterpret_cast<uint32_t *>(host + off_first);
    merge.q_rows = sessions[0].q_rows;
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
        h_merge[i].out = s.out; h_merge[i].q_rows = s.q_rows; h_first[i] = total_rows;
        if (s.q_rows != merge.q_rows) merge.q_rows = 0;
        TTDecodeSession &d = tmp[i];
        d.q = s.q; d.out = s.out; d.k = s.k; d.v = s.v; d.seq_len = s.seq_len; d.q_rows = s.q_rows; d.kv_start = 0;
        d.n_parts = 0; d.partial_base = 0; d.ring_capacity = 0; d.keep = nullptr; d.row_index = nullptr;
        total_rows += s.q_rows;
    }
    const uint32_t n_table = fused ? n_groups + n_sessions : n_groups;
    uint32_t fused_lens[GROUPS], fused_rows[GROUPS];
    uint32_t *lens = fused ? fused_lens : ctx->h_prefix_lens, *rows = fused ? fused_rows : ctx->h_prefix_rows;
    for (uint32_t g = 0, first = 0; g < n_groups; ++g) {
        lens[g] = groups[g].prefix_len;
        rows[g] = 0;
        for (uint32_t i = 0; i < groups[g].n_sessions; ++i) rows[g] += sessions[first + i].q_rows;
        first += groups[g].n_sessions;
    }
    if (fused) {
        if (q.io_dtype != TT_F16 && q.io_dtype != TT_BF16) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "io_dtype must be TT_F16 or TT_BF16");
        if (q.q_row_stride_elements < q.n_q_heads * q.head_dim || q.out_row_stride_elements < q.n_q_heads * q.head_dim)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "a row stride is smaller than its tight width");
        if (q.q_row_stride_elements % 8 || q.out_row_stride_elements % 4)
            return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "row strides must keep rows 16-byte aligned");
        for (uint32_t i = 0; i < n_sessions; ++i) {
            if (sessions[i].k == nullptr || sessions[i].v == nullptr) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u has a null buffer", i);
            if (((uintptr_t)sessions[i].k | (uintptr_t)sessions[i].v) & 15)
                return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "session %u: buffers must be 16-byte aligned", i);
            lens[n_groups + i] = sessions[i].seq_len;
            rows[n_groups + i] = sessions[i].q_rows;
        }
    }
    // ---- plan: the prefix pass may take half of the workspace, at its end ----
    uint32_t keys_per_item = 0, n_items = 0;
    const size_t room = ctx->workspace_bytes / 2;
    if (tt_attn_plan_prefix_splits(lens, rows, n_table, q.head_dim, q.n_q_heads, q.n_kv_heads, (uint32_t)ctx->sm_count, room,
                                   &keys_per_item, &n_items) != TT_OK)
        return tt_set_error(ctx, TT_ERR_OOM, "the prefix partials do not fit the context workspace");
    const uint32_t group = q.n_q_heads / q.n_kv_heads, tile_rows = rows_per_tile(rows, n_table, group, q.head_dim);
    uint32_t item = 0, partial = 0;
    // group g of the table: `len` keys at k, v for the query rows of sessions first .. first + count - 1
    auto add_group = [&](uint32_t g, const void *k, const void *v, uint32_t first, uint32_t count, bool own) {
        PrefixGroup &d = h_groups[g];
        d.prefix_len = lens[g];
        d.n_parts = ceil_div(lens[g], keys_per_item);
        d.part_len = keys_per_item;
        if (d.n_parts != 0) {               // parts of equal length
            d.part_len = ceil_div(ceil_div(lens[g], d.n_parts), kBK) * kBK;
            d.n_parts = ceil_div(lens[g], d.part_len);
        }
        d.session_begin = first; d.session_count = count;
        d.row_begin = h_first[first]; d.n_rows = rows[g];
        d.partial_base = partial; d.item_begin = item;
        if (in_params) table.item_begin[g] = item;
        d.row_tiles = ceil_div((uint64_t)rows[g] * group, tile_rows);
        d.q = sessions[first].q; d.q_rows = sessions[first].q_rows; d.q_step = 0;
        if (count > 1) d.q_step = (long long)((uintptr_t)sessions[first + 1].q - (uintptr_t)sessions[first].q);
        for (uint32_t i = 1; i < count; ++i)
            if (sessions[first + i].q_rows != d.q_rows ||
                (long long)((uintptr_t)sessions[first + i].q - (uintptr_t)sessions[first + i - 1].q) != d.q_step) d.q_rows = 0;
        d.causal_rows = own ? rows[g] : 0u;
        d.pad = 0;
        for (uint32_t i = 0; i < count; ++i) {
            MergeSession &m = h_merge[first + i];
            if (own) {
                m.own_base = partial;
                m.own_parts = d.n_parts;
            } else {
                m.prefix_base = partial + (h_first[first + i] - d.row_begin) * q.n_q_heads;
                m.prefix_parts = d.n_parts;
                m.prefix_stride = rows[g] * q.n_q_heads;
            }
        }
        item += d.n_parts * q.n_kv_heads * d.row_tiles;
        partial += d.n_parts * rows[g] * q.n_q_heads;
        const uint64_t width = (uint64_t)q.n_kv_heads * q.head_dim;
        return lens[g] == 0 ||
               (tt_make_tensor_map_2d(reinterpret_cast<CUtensorMap *>(h_maps[g].m[0]), k, q.io_dtype, width, lens[g], q.kv_token_stride_elements, 64) &&
                tt_make_tensor_map_2d(reinterpret_cast<CUtensorMap *>(h_maps[g].m[1]), v, q.io_dtype, width, lens[g], q.kv_token_stride_elements, 64));
    };
    bool encoded = true;
    for (uint32_t g = 0, first = 0; g < n_groups; ++g) {
        encoded = encoded && add_group(g, groups[g].k, groups[g].v, first, groups[g].n_sessions, false);
        first += groups[g].n_sessions;
    }
    if (fused) {        // the longest sessions first: what starts last is short
        uint32_t order[kFusedSessions];
        for (uint32_t i = 0; i < n_sessions; ++i) {
            uint32_t at = i;
            for (; at > 0 && sessions[order[at - 1]].seq_len < sessions[i].seq_len; --at) order[at] = order[at - 1];
            order[at] = i;
        }
        for (uint32_t i = 0; i < n_sessions; ++i) {
            const uint32_t x = order[i];
            lens[n_groups + i] = sessions[x].seq_len;
            rows[n_groups + i] = sessions[x].q_rows;
            encoded = encoded && add_group(n_groups + i, sessions[x].k, sessions[x].v, x, 1, true);
        }
    }
    if (!encoded) return tt_set_error(ctx, TT_ERR_CUDA, "cuTensorMapEncodeTiled failed for the prefix operands");
    const size_t partial_bytes = ((size_t)partial * (q.head_dim + 2) * sizeof(float) + 255) / 256 * 256;
    kp.part_o = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->partials) + (ctx->workspace_bytes / 256 * 256 - partial_bytes));
    kp.part_m = kp.part_o + (size_t)partial * q.head_dim;
    kp.part_l = kp.part_m + partial;

    // ---- suffix pass (it also checks the rest of the arguments) ----
    TTDecodeForm own;
    if (fused) {
        own.part_o = kp.part_o; own.part_m = kp.part_m; own.part_l = kp.part_l;
    } else {
        own.reserved_bytes = partial_bytes + 256;
        own.partials_only = true;
        own.short_sessions = true;
        const int rc = tt_launch_decode(ctx, (cudaStream_t)stream, tmp, n_sessions, params, 0, nullptr, nullptr, nullptr, nullptr, nullptr, &own);
        if (rc != TT_OK) return rc;
        for (uint32_t i = 0; i < n_sessions; ++i) {
            h_merge[i].own_base = ctx->h_sessions[i].partial_base;
            h_merge[i].own_parts = ctx->h_sessions[i].n_parts;
        }
    }
    cudaError_t e = cudaSuccess;
    if (!in_params) {
        e = cudaMemcpyAsync(ctx->prefix_tables, host, table_bytes, cudaMemcpyHostToDevice, (cudaStream_t)stream);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "copy prefix tables");
    }
    // ---- prefix pass ----
    kp.maps = reinterpret_cast<const PrefixMaps *>(ctx->prefix_tables);
    kp.groups = reinterpret_cast<const PrefixGroup *>(ctx->prefix_tables + off_groups);
    kp.sessions = reinterpret_cast<const PrefixSession *>(ctx->prefix_tables + off_sessions);
    kp.n_q_heads = q.n_q_heads; kp.n_kv_heads = q.n_kv_heads; kp.q_row_stride = q.q_row_stride_elements;
    kp.behind_own_rows = fused ? 0u : 1u;
    table.n_groups = n_table; table.n_sessions = n_sessions; table.in_params = in_params ? 1u : 0u;
    merge.n = in_params ? n_sessions : 0u;
    if (item != 0) {
        const RowsParams rp = tile_rows == 256 ? pair_params(q.scale, q.io_dtype) : rows_params(q.scale, q.io_dtype, q.head_dim);
        e = q.io_dtype == TT_F16 ? launch_prefix<__half>((cudaStream_t)stream, q.head_dim, tile_rows, item, rp, ctx->status, kp)
                                 : launch_prefix<__nv_bfloat16>((cudaStream_t)stream, q.head_dim, tile_rows, item, rp, ctx->status, kp);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_prefix launch");
        ctx->launches++;
    }
    // ---- merge ----
    uint32_t parts = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) parts = std::max(parts, h_merge[i].prefix_parts + h_merge[i].own_parts);
    const MergeSession *dev = reinterpret_cast<const MergeSession *>(ctx->prefix_tables + off_merge);
    const uint32_t *dev_first = reinterpret_cast<const uint32_t *>(ctx->prefix_tables + off_first);
    e = q.io_dtype == TT_F16
            ? launch_merge<__half>((cudaStream_t)stream, q.head_dim, total_rows * q.n_q_heads, parts, merge, dev, dev_first, n_sessions, kp, own, q.n_q_heads, q.out_row_stride_elements, (uint32_t)ctx->sm_count)
            : launch_merge<__nv_bfloat16>((cudaStream_t)stream, q.head_dim, total_rows * q.n_q_heads, parts, merge, dev, dev_first, n_sessions, kp, own, q.n_q_heads, q.out_row_stride_elements, (uint32_t)ctx->sm_count);
    if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_prefix_merge launch");
    ctx->launches++;
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
    // The sessions' own rows as groups of one session each in the prefix pass: one launch less, no second pass that starts
    // when the first one ends, and the tensor cores for draft rows. Us a call with a pass of their own, then so:
    //   more than the 16 packed rows a split-KV item takes, up to 64 sessions (whose maps and groups make the parameters 25 KB,
    //     8 us more of host time than 16 sessions): 16 sessions of 4 rows of 16 heads 176, 82; 64 of 4 rows and 800 to 1600
    //     keys 220, 123, of 4 to 300 98, 94;
    //   head_dim 256: up to 16 sessions (4 of short keys 18.5, 13; 16 of 4000 to 8000 46, 43, with 8 KV heads 122, 118), and up to
    //     32 where items of 128 rows do (8 KV heads, 32 of 1 to 1024 keys 42, 44, of 1024 to 32768 389, 380) but not of 256 (2
    //     KV heads, 32 of 4000 to 8000 76, 101);
    //   head_dim 64 and 128: up to 32 sessions whose streams, one a KV head, leave half of the SMs free (128, 2 KV heads, 32 of
    //     800 to 1600 keys 26, 19; 8 KV heads, 8 of 4000 to 8000 69, 45, but 10 50, 56 and 24 100, 130; 64, 8 KV heads, 8 33,
    //     20, 24 of 800 to 1600 25, 31), or up to one an SM of at most 1024 keys (4 KV heads, 24 20.5, 19.0; 8, 16 20.3, 21.0, of 64 17.8, 16.5).
    bool fused = false;
    if (in_params) {
        uint32_t group_rows = 0, most_rows = 0, most_own = 0, longest = 0;
        for (uint32_t g = 0, i = 0; g < n_groups; ++g, group_rows = 0)
            for (uint32_t x = 0; x < groups[g].n_sessions; ++x, ++i) {
                group_rows += sessions[i].q_rows;
                most_rows = std::max(most_rows, group_rows);
                most_own = std::max(most_own, sessions[i].q_rows);
                longest = std::max(longest, sessions[i].seq_len);
            }
        const uint32_t heads = q.n_q_heads / q.n_kv_heads, sms = (uint32_t)ctx->sm_count;
        const uint64_t streams = (uint64_t)n_sessions * q.n_kv_heads;
        fused = most_own * heads > 16 ? true
                : q.head_dim == 256 ? n_sessions <= 16 || (n_sessions <= 32 && rows_per_tile(&most_rows, 1, heads, q.head_dim) < 256)
                                    : n_sessions <= 32 && (streams * 2 <= sms || (streams <= sms && longest <= 1024));
    }
    return !in_params || n_groups + (fused ? n_sessions : 0u) <= kFewGroups
               ? shared_prefix<kFewGroups>(ctx, stream, groups, n_groups, sessions, n_sessions, params, in_params, fused)
               : shared_prefix<kTableGroups>(ctx, stream, groups, n_groups, sessions, n_sessions, params, in_params, fused);
}

// Whether the tensor cores take a sink call: more packed rows than a split-KV item has (which reads K and V again for every
// 16 of them; 16 sessions of 4 rows of 8 heads, 1024 keys: 25.2 us against 14.9, 4096 keys 70 against 34; of 16 heads 143 against
// 35). Sessions beyond one launch's tables need more than a tile or two of keys (64 sessions of 64 keys,
// head_dim 128: 13.9 us in clusters, 20.5 here; of 1024 62 and 31).
bool tt_sink_rows_form(const TTDecodeSession *sessions, uint32_t n_sessions, const tt_attn_batch_params *p) {
    if (!(p->scale > 0.f)) return false;
    uint32_t most_rows = 0, most_keys = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        most_rows = std::max(most_rows, sessions[i].q_rows);
        most_keys = std::max(most_keys, sessions[i].seq_len - std::min(sessions[i].seq_len, sessions[i].kv_start));
    }
    return most_rows * (p->n_q_heads / p->n_kv_heads) > 16 && (n_sessions <= SinkRowsForm<kTableGroups>::kSessions || most_keys > 2 * kBK);
}

// One launch and merge of that form.
template <uint32_t GROUPS>
static int launch_sink_rows(tt_context *ctx, cudaStream_t stream, const TTDecodeSession *sessions, uint32_t n_sessions, const TTDecodeForm &form,
                            const tt_attn_batch_params *p) {
    const tt_attn_batch_params &q = *p;
    const uint32_t group = q.n_q_heads / q.n_kv_heads;
    using Form = SinkRowsForm<GROUPS>;
    constexpr uint32_t kSessions = Form::kSessions;
    static thread_local Form f;
    static thread_local MergeTable merge;
    f.n_q_heads = q.n_q_heads; f.n_kv_heads = q.n_kv_heads; f.q_row_stride = q.q_row_stride_elements; f.behind_own_rows = 0;
    f.groups = nullptr; f.sessions = nullptr; f.maps = nullptr;
    f.sink = form.sink; f.window = form.window;
    f.table.n_groups = n_sessions; f.table.n_sessions = n_sessions; f.table.in_params = 1;
    merge.n = n_sessions; merge.q_rows = sessions[0].q_rows;
    // the longest first
    uint32_t order[kSessions] = {}, keys[kSessions] = {}, lens[kSessions] = {}, rows[kSessions] = {}, total_rows = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        const TTDecodeSession &s = sessions[i];
        typename Form::Session &d = f.session[i];
        d.seq_len = s.seq_len; d.q_rows = s.q_rows;
        d.windowed = s.seq_len > form.window && s.seq_len - form.window > form.sink ? 1u : 0u;
        d.base = d.windowed ? s.kv_start : 0u;
        d.first_row = d.base;
        d.straight = s.seq_len - d.base;
        if (s.ring_capacity != 0 && s.seq_len > (uint64_t)form.sink + s.ring_capacity) {        // wrapped, hence windowed
            d.first_row = form.sink + (d.base - form.sink) % s.ring_capacity;
            d.straight = std::min(d.straight, form.sink + s.ring_capacity - d.first_row);
        }
        const uint32_t behind = s.seq_len - d.base - d.straight;
        keys[i] = (d.windowed ? (form.sink + 63) / 64 * 64 : 0u) + (behind != 0 ? (d.straight + 63) / 64 * 64 + behind : d.straight);
        f.table.s[i].q = s.q; f.table.s[i].first_row = total_rows; f.table.s[i].q_rows = s.q_rows;
        merge.first_row[i] = total_rows;
        MergeSession &m = merge.s[i];
        m.out = s.out; m.q_rows = s.q_rows; m.prefix_base = 0; m.prefix_parts = 0; m.prefix_stride = 0;
        if (s.q_rows != merge.q_rows) merge.q_rows = 0;
        total_rows += s.q_rows;
        uint32_t at = i;
        for (; at > 0 && keys[order[at - 1]] < keys[i]; --at) order[at] = order[at - 1];
        order[at] = i;
    }
    for (uint32_t g = 0; g < n_sessions; ++g) { lens[g] = keys[order[g]]; rows[g] = sessions[order[g]].q_rows; }
    uint32_t keys_per_item = 0, n_items = 0, item = 0, partial = 0, parts = 0;
    if (tt_attn_plan_prefix_splits(lens, rows, n_sessions, q.head_dim, q.n_q_heads, q.n_kv_heads, (uint32_t)ctx->sm_count, ctx->workspace_bytes,
                                   &keys_per_item, &n_items) != TT_OK)
        return tt_set_error(ctx, TT_ERR_OOM, "the partials do not fit the context workspace");
    const uint32_t tile_rows = rows_per_tile(rows, n_sessions, group, q.head_dim);
    const uint64_t width = (uint64_t)q.n_kv_heads * q.head_dim;
    for (uint32_t g = 0; g < n_sessions; ++g) {
        const uint32_t x = order[g];
        const TTDecodeSession &s = sessions[x];
        PrefixGroup &d = f.table.g[g];
        d.prefix_len = lens[g];
        d.n_parts = ceil_div(lens[g], keys_per_item);
        d.part_len = d.n_parts != 0 ? ceil_div(ceil_div(lens[g], d.n_parts), kBK) * kBK : keys_per_item;
        if (d.n_parts != 0) d.n_parts = ceil_div(lens[g], d.part_len);       // parts of equal length
        d.session_begin = x; d.session_count = 1;
        d.row_begin = merge.first_row[x]; d.n_rows = s.q_rows;
        d.partial_base = partial; d.item_begin = item;
        f.table.item_begin[g] = item;
        d.row_tiles = ceil_div((uint64_t)s.q_rows * group, tile_rows);
        d.q = s.q; d.q_rows = s.q_rows; d.q_step = 0; d.causal_rows = s.q_rows; d.pad = 0;
        merge.s[x].own_base = partial; merge.s[x].own_parts = d.n_parts;
        item += d.n_parts * q.n_kv_heads * d.row_tiles;
        partial += d.n_parts * s.q_rows * q.n_q_heads;
        parts = std::max(parts, d.n_parts);
        if (lens[g] == 0) continue;
        const typename Form::Session &e = f.session[x];
        const uint64_t cached = s.ring_capacity != 0 ? std::min<uint64_t>(s.seq_len, (uint64_t)form.sink + s.ring_capacity) : s.seq_len;
        const uint64_t sinks = std::max<uint64_t>(1, std::min<uint64_t>(form.sink, cached));
        const uint64_t behind = form.sink + (uint64_t)(s.seq_len - e.base - e.straight);
        auto encode = [&](unsigned char *map, const void *from, uint64_t count) {
            return tt_make_tensor_map_2d(reinterpret_cast<CUtensorMap *>(map), from, q.io_dtype, width, count, q.kv_token_stride_elements, 64);
        };
        if (!encode(f.table.maps[g].m[0], s.k, cached) || !encode(f.table.maps[g].m[1], s.v, (uint64_t)e.first_row + e.straight) ||
            !encode(f.table.maps[kSessions + x].m[0], s.v, sinks) ||
            !encode(f.table.maps[kSessions + x].m[1], s.v, std::max<uint64_t>(1, std::min(behind, cached))))
            return tt_set_error(ctx, TT_ERR_CUDA, "cuTensorMapEncodeTiled failed for the decode operands");
    }
    f.part_o = ctx->partials; f.part_m = f.part_o + (size_t)partial * q.head_dim; f.part_l = f.part_m + partial;
    cudaError_t e = cudaSuccess;
    if (item != 0) {
        const RowsParams rp = tile_rows == 256 ? pair_params(q.scale, q.io_dtype) : rows_params(q.scale, q.io_dtype, q.head_dim);
        TTLaunchTimer timer(ctx, stream, TT_PROFILE_DECODE_PARTIAL);
        e = q.io_dtype == TT_F16 ? launch_prefix<__half>(stream, q.head_dim, tile_rows, item, rp, ctx->status, f)
                                 : launch_prefix<__nv_bfloat16>(stream, q.head_dim, tile_rows, item, rp, ctx->status, f);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_sink launch");
        timer.stop();
        ctx->launches++;
    }
    TTDecodeForm own;
    own.part_o = f.part_o; own.part_m = f.part_m; own.part_l = f.part_l;
    const uint32_t out_rows = total_rows * q.n_q_heads;
    e = q.io_dtype == TT_F16 ? launch_merge<__half>(stream, q.head_dim, out_rows, parts, merge, nullptr, nullptr, n_sessions, f, own, q.n_q_heads,
                                                    q.out_row_stride_elements, (uint32_t)ctx->sm_count)
                             : launch_merge<__nv_bfloat16>(stream, q.head_dim, out_rows, parts, merge, nullptr, nullptr, n_sessions, f, own, q.n_q_heads,
                                                           q.out_row_stride_elements, (uint32_t)ctx->sm_count);
    if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_sink merge launch");
    ctx->launches++;
    return TT_OK;
}

// Launches the form for sessions checked by tt_launch_decode, as many at a time as the parameters take; kv_start is the first key
// of the rows' windows behind the sinks.
int tt_launch_sink_rows(tt_context *ctx, cudaStream_t stream, const TTDecodeSession *sessions, uint32_t n_sessions, const TTDecodeForm &form,
                        const tt_attn_batch_params *p) {
    const uint32_t passes = ceil_div(n_sessions, SinkRowsForm<kTableGroups>::kSessions), each = ceil_div(n_sessions, passes);
    for (uint32_t i = 0; i < n_sessions; i += each) {
        const uint32_t n = std::min(each, n_sessions - i);
        const int rc = n <= SinkRowsForm<kFewGroups>::kSessions ? launch_sink_rows<kFewGroups>(ctx, stream, sessions + i, n, form, p)
                                                               : launch_sink_rows<kTableGroups>(ctx, stream, sessions + i, n, form, p);
        if (rc != TT_OK) return rc;
    }
    return TT_OK;
}
