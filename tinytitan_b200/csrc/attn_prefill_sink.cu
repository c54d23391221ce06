// Prefill over the first tokens and a sliding window on the sm_100a tensor cores, head_dim 256.
//
// Query t of a chunk (position start + t) sees key j when j <= start + t and (j < sink or j > start + t - window). An
// item of attn_pair_kernel (attn_pair_tc.cuh) is 256 rows: all heads of a KV head, or the largest power of two that divides
// their number, times consecutive queries. Its keys are the window of its queries, window + queries - 1 of them, so few queries
// of many heads leave less that only some rows see (8192 tokens, 8 heads per KV head, window 2048: 212 us with 8 heads x 32
// queries, 217 with 4 x 64, 224 with 2 x 128).
//
// When the window of an item's last query starts behind the sinks, its keys are the halves of 64 keys over [0, sink), read
// through tensor maps that end with the sinks, and then those from the first query's window start on: what lies between
// is neither read nor counted, and may hold anything. A tile is two halves, which need not be neighbours. Otherwise the
// halves start at key 0 and every key up to the last query's own is visible to that query. In a ring cache the window's
// halves start at a multiple of 64 rows of the ring, so that no box runs over the ring's end; rows that a query does not
// see are masked by their logical position.
//
// An item is short, so what it costs besides its tiles shows: Q arrives as whole rows by asynchronous copies while the
// first K and V chunks are in flight, and the output leaves as whole rows.
#include "attn_pair_tc.cuh"

namespace {

constexpr uint32_t kBoxKeys = 64;
constexpr uint32_t kMaxHeadBits = 5;     // at least 8 queries of a head

struct alignas(64) SinkForm {
    static constexpr bool kPartials = false;
    CUtensorMap k_map, v_map;            // all rows, boxes of 64 keys
    CUtensorMap k_sink, v_sink;          // rows [0, sink) alone: the rest of a tile reads as zeros
    const unsigned char *q;
    unsigned char *out;
    uint32_t start_position, query_count, n_q_heads, n_kv_heads, kv_valid_count, window;   // window >= 1
    uint32_t q_stride, o_stride;         // elements
    uint32_t sink, ring;                 // ring: a multiple of 64, 0 = plain rows
    uint32_t n_q_tiles, head_bits;       // an item: 256 >> head_bits queries of 1 << head_bits adjacent q heads of one KV head

    struct Item : RowsItem {
        uint32_t head, row0;             // first q head, first query
        uint32_t queries;
        uint32_t sink_halves;            // halves over [0, sink) before the window's
        uint32_t base;                   // first key of the window's halves
        uint32_t base_row;               // ... and its cache row behind the sinks, in a ring
        bool windowed;                   // some query's window starts behind the sinks
    };
    __device__ __forceinline__ Item item(uint32_t block, int hd, int rows) const {
        Item it;
        // long items (late queries) first; the heads of one KV group are adjacent and share their keys in L2
        const uint32_t units = n_q_heads >> head_bits, tile_queries = 256u >> head_bits;
        it.head = block % units << head_bits;
        it.kv_head = it.head / (n_q_heads / n_kv_heads);
        it.row0 = (n_q_tiles - 1 - block / units) * tile_queries;
        it.queries = min(tile_queries, query_count - it.row0);
        const uint32_t first = start_position + it.row0, last = first + it.queries - 1;  // positions of the first and last query
        const uint32_t key_end = min(kv_valid_count, last + 1);
        it.sink_halves = 0; it.base = 0;
        it.windowed = last + 1 > window && last + 1 - window > sink;
        if (it.windowed) {
            const uint32_t from = first + 1 > window ? first + 1 - window : 0u;
            it.sink_halves = (sink + kBoxKeys - 1) / kBoxKeys;
            it.base = max(sink, from);
            if (ring) it.base = sink + (it.base - sink) / kBoxKeys * kBoxKeys;
        }
        it.base_row = ring && it.windowed ? (it.base - sink) % ring : 0u;
        it.n_halves = it.sink_halves + (key_end - it.base + kBoxKeys - 1) / kBoxKeys;
        it.n_tiles = (it.n_halves + 1) / 2;
        return it;
    }
    // row r of an item: query r % tile_queries of head r / tile_queries
    __device__ __forceinline__ uint32_t query_of(uint32_t r) const { return r & ((256u >> head_bits) - 1); }
    __device__ __forceinline__ uint32_t head_of(const Item &it, uint32_t r) const { return it.head + (r >> (8 - head_bits)); }
    __device__ __forceinline__ const void *query(const Item &it, uint32_t r, int hd, int rows) const {
        const uint32_t t = query_of(r);
        return t < it.queries ? q + ((size_t)(it.row0 + t) * q_stride + (size_t)head_of(it, r) * hd) * 2 : nullptr;
    }
    __device__ __forceinline__ void acquire(const Item &) const {}
    __device__ __forceinline__ bool waits_late() const { return false; }
    __device__ __forceinline__ const CUtensorMap *box(const Item &it, uint32_t tile, uint32_t half, bool is_k, int &row) const {
        const uint32_t u = 2 * tile + half;
        if (u < it.sink_halves) {
            row = (int)(u * kBoxKeys);
            return is_k ? &k_sink : &v_sink;
        }
        uint32_t off = (u - it.sink_halves) * kBoxKeys;
        if (ring && it.windowed) {
            off += it.base_row;
            while (off >= ring) off -= ring;
            row = (int)(sink + off);
        } else {
            row = (int)(it.base + off);
        }
        return is_k ? &k_map : &v_map;
    }
    __device__ __forceinline__ bool masked(const Item &it, uint32_t tile) const {
        if (2 * tile < it.sink_halves) return true;
        const uint32_t key0 = it.base + (2 * tile - it.sink_halves) * kBoxKeys, first = start_position + it.row0, last = first + it.queries - 1;
        return key0 + kBK > min(kv_valid_count, first + 1) || (it.windowed && last + 1 > window && key0 < max(sink, last + 1 - window));
    }
    __device__ __forceinline__ void visible(const Item &it, uint32_t row, uint32_t tile, uint32_t (&bits)[4]) const {
        const uint32_t at = start_position + it.row0 + query_of(row), end = min(kv_valid_count, at + 1);
        // when no window starts behind the sinks the halves start at key 0, and every query's window reaches back to the sinks
        const uint32_t from = it.windowed ? max(sink, at + 1 > window ? at + 1 - window : 0u) : 0u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t u = 2 * tile + half;
            const bool of_sink = u < it.sink_halves;
            const int key0 = (int)(of_sink ? u * kBoxKeys : it.base + (u - it.sink_halves) * kBoxKeys);
            const int lo = of_sink ? 0 : (int)from - key0, hi = (int)(of_sink ? min(end, sink) : end) - key0;
            bits[2 * half] = bits_between(lo, hi);
            bits[2 * half + 1] = bits_between(lo - 32, hi - 32);
        }
    }
    __device__ __forceinline__ bool exists(const Item &it, uint32_t r) const { return query_of(r) < it.queries; }
    __device__ __forceinline__ void *output(const Item &it, uint32_t r, int hd) const {
        return out + ((size_t)(it.row0 + query_of(r)) * o_stride + (size_t)head_of(it, r) * hd) * 2;
    }
};

}  // namespace

int tt_launch_prefill_sink(tt_context *ctx, cudaStream_t stream, const void *q, const void *k, const void *v, void *out,
                           const tt_prefill_params *p, uint32_t io_dtype, uint32_t sink_tokens, uint32_t ring) {
    const uint64_t width = (uint64_t)p->n_kv_heads * 256;
    uint64_t rows = p->kv_valid_count;
    if (ring != 0 && rows > (uint64_t)sink_tokens + ring) rows = (uint64_t)sink_tokens + ring;
    const uint64_t sink_rows = sink_tokens == 0 ? 1 : sink_tokens < rows ? sink_tokens : rows;
    SinkForm f;
    if (!tt_make_tensor_map_2d(&f.k_map, k, io_dtype, width, rows, p->kv_token_stride_elements, kBoxKeys) ||
        !tt_make_tensor_map_2d(&f.v_map, v, io_dtype, width, rows, p->kv_token_stride_elements, kBoxKeys) ||
        !tt_make_tensor_map_2d(&f.k_sink, k, io_dtype, width, sink_rows, p->kv_token_stride_elements, kBoxKeys) ||
        !tt_make_tensor_map_2d(&f.v_sink, v, io_dtype, width, sink_rows, p->kv_token_stride_elements, kBoxKeys))
        return tt_set_error(ctx, TT_ERR_CUDA, "cuTensorMapEncodeTiled failed for the prefill operands");
    f.q = (const unsigned char *)q; f.out = (unsigned char *)out;
    f.start_position = p->start_position; f.query_count = p->query_count; f.n_q_heads = p->n_q_heads; f.n_kv_heads = p->n_kv_heads;
    f.kv_valid_count = p->kv_valid_count;
    f.window = p->sliding_window == 0 ? UINT32_MAX : p->sliding_window;
    f.q_stride = p->q_token_stride_elements; f.o_stride = p->o_token_stride_elements;
    f.sink = sink_tokens; f.ring = ring;
    uint32_t head_bits = 0;
    while (head_bits < kMaxHeadBits && (p->n_q_heads / p->n_kv_heads >> head_bits) % 2 == 0) ++head_bits;
    f.head_bits = head_bits;
    f.n_q_tiles = (p->query_count + (256u >> head_bits) - 1) / (256u >> head_bits);
    const RowsParams rp = pair_params(p->scale, io_dtype);
    const uint32_t items = f.n_q_tiles * (p->n_q_heads >> head_bits);
    const cudaError_t e = io_dtype == TT_F16 ? launch_pair<__half>(stream, items, rp, ctx->status, f)
                                             : launch_pair<__nv_bfloat16>(stream, items, rp, ctx->status, f);
    if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_prefill_sink launch");
    ctx->launches++;
    return TT_OK;
}
