// Decode attention over the first tokens and a sliding window ("sinks"), batched over sessions.
//
// The reference's sliding-window decode (Attention.encodeSWA,
// sources/TinyTitan/Kernels/Attention/Attention.swift:233-266) forgets everything before the window. Softmax
// weights sum to one, so heads that have nothing to attend to put their weight on the first tokens, and a model
// whose first tokens are evicted loses its footing; keeping a few of them visible next to the window restores it
// and bounds an endless session's cache at sink + window rows.
//
// Row r of a session's W rows (end_r = seq_len - (W - 1 - r)) sees key j when j < end_r and (j < sink or
// j >= end_r - window). It reads the union of its rows' keys once per KV head and nothing else, in the split-KV
// pass 1 of the decode kernel (attn_pass1.cuh): that kernel fetches single cache rows, so skipping from the sinks to
// the window and wrapping around a ring cost an address each, no tile is half empty, and its bound stays the bytes of
// the visible rows. With one row every fetched key is visible and no score is masked. A window bounds the keys of a
// session, so its parts often fit one cluster of CTAs, which joins them without the partials and the second launch that
// unbounded decode needs; draft rows beyond a split-KV item's 16 go to the tensor cores (tt_sink_rows_form). 32 sessions of up to 4100 keys, 16/2 heads of 256: 46 us, 5.8 TB/s; one of 1024 keys 8.9 us.
#include "attn_pass1.cuh"

cudaError_t tt_launch_pass1_sink(cudaStream_t stream, uint32_t n_items, const TTDecodeItem *items, const TTDecodeSession *sessions,
                                 const TTDecodeForm &form, const tt_attn_batch_params *p, uint32_t *status,
                                 const TTSessionTable &table, uint32_t table_keys, bool wide_rows, uint32_t hpc) {
    PassExtra<kPassSink> extra;
    extra.sink = form.sink;
    extra.window = form.window;
    if (p->io_dtype == TT_F16)
        return launch_partial_hd<__half>(stream, n_items, items, sessions, form.part_o, form.part_m, form.part_l, p, status,
                                         table, table_keys, wide_rows, hpc, extra);
    return launch_partial_hd<__nv_bfloat16>(stream, n_items, items, sessions, form.part_o, form.part_m, form.part_l, p, status,
                                            table, table_keys, wide_rows, hpc, extra);
}

namespace {

cudaError_t launch_cluster(cudaStream_t stream, uint32_t n_ctas, const PassExtra<kPassSinkCluster> &extra, const tt_attn_batch_params *p,
                           uint32_t *status, const TTSessionTable &table, bool wide_rows, uint32_t hpc) {
    if (p->io_dtype == TT_F16)
        return launch_partial_hd<__half>(stream, n_ctas, nullptr, nullptr, nullptr, nullptr, nullptr, p, status, table, 0, wide_rows, hpc, extra);
    return launch_partial_hd<__nv_bfloat16>(stream, n_ctas, nullptr, nullptr, nullptr, nullptr, nullptr, p, status, table, 0, wide_rows, hpc, extra);
}

// Clusters of 1 << bits CTAs of the kernel for `p` that run at once: asked once per kernel and context, a query is some
// microseconds.
uint32_t resident_clusters(tt_context *ctx, const tt_attn_batch_params *p, bool wide_rows, uint32_t hpc, uint32_t bits) {
    const uint32_t kernel = (p->head_dim >> 7) * 8 + (p->io_dtype == TT_F16 ? 4 : 0) + (wide_rows ? 2 : 0) + (hpc == 2 ? 1 : 0);   // 64, 128, 256: 0, 1, 2
    int &known = ctx->sink_clusters[kernel][bits];
    if (known == 0) {
        int n = 0;
        PassExtra<kPassSinkCluster> extra = {};
        extra.cluster = 1u << bits;
        extra.resident = &n;
        if (launch_cluster(nullptr, 1u << bits, extra, p, nullptr, ctx->session_table, wide_rows, hpc) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        known = n > 0 ? n : -1;
    }
    return known > 0 ? (uint32_t)known : 0u;
}

}  // namespace

// One launch instead of two where the parts of a (session, KV heads, row tile) -- a stream -- can be one cluster. It is
// taken with the largest clusters of which all streams' run at once,
//   when a CTA has at most 64 keys (32 with two n-tiles of query rows), for latency: 1 session of 1024 keys, head_dim 256,
//   8.3 us against 9.8; of 2048, 13.4 against 9.8;
//   when the clusters fill the machine with sessions of one length, for then no CTA waits for another: 32 sessions of 4096
//   keys 45.7 us against 48.9, 64 of 2048 46.2 against 52.1, at head_dim 128 with 8 KV heads 32 of 1024 26.2 against 38.5.
//   A half-empty machine is left to finer parts (16 of 4096: 44.1 us against 26.8), and so are more than 1024 keys a CTA (256
//   with two n-tiles: 16 sessions of 4 rows and 4096 keys 74.7 us against 70.2).
// Draft rows that the tensor-core form takes (tt_sink_rows_form) are left to it except for the latency of short ones on half a
// machine (2 sessions of 4 rows of 8 heads, 256 keys: 8.8 us against 11.4).
// 0: the parts meet through memory in a second launch.
static uint32_t cluster_size(tt_context *ctx, const uint32_t *keys, uint32_t n_sessions, const tt_attn_batch_params *p, uint64_t streams,
                             bool wide_rows, uint32_t hpc, bool rows_form) {
    uint64_t longest = 0, sum = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        longest = keys[i] > longest ? keys[i] : longest;
        sum += keys[i];
    }
    uint32_t bits = 0;
    while ((kMaxSinkCluster >> (bits + 1)) != 0 && (uint64_t)(kKeysPerBlock << bits) < longest) ++bits;
    uint32_t resident = resident_clusters(ctx, p, wide_rows, hpc, bits);
    // clusters of 16 as long as they have room: 31 of 32 keys a CTA on 32 places 13.5 us, as two of eight CTAs 10
    while (bits > 0 && streams * (bits == 4 ? 2 : 1) > resident) resident = resident_clusters(ctx, p, wide_rows, hpc, --bits);
    if (streams > resident) return 0;
    const uint64_t per_cta = (longest + (1u << bits) - 1) >> bits;
    const uint64_t ctas = streams << bits, machine = resident_clusters(ctx, p, wide_rows, hpc, 0);
    if (rows_form) return per_cta <= 32 && ctas * 2 <= machine ? 1u << bits : 0u;
    if (per_cta <= (wide_rows ? 32u : 64u)) return 1u << bits;
    const bool full = ctas * 6 >= machine * 5;
    return full && per_cta <= (wide_rows ? 256u : 1024u) && sum * 128 >= longest * n_sessions * 127 ? 1u << bits : 0u;
}

// Launches the cluster form when it is the faster one; *taken says whether.
int tt_launch_sink_cluster(tt_context *ctx, cudaStream_t stream, const TTDecodeSession *sessions, const uint32_t *keys, uint32_t n_sessions,
                           const TTDecodeForm &form, const tt_attn_batch_params *p, uint32_t hpc, bool rows_form, bool *taken) {
    const uint32_t group = p->n_q_heads / p->n_kv_heads;
    auto row_tiles = [&](uint32_t i) { return (sessions[i].q_rows * group + 15) / 16; };
    uint64_t streams = 0;
    bool wide_rows = false;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        streams += (uint64_t)(p->n_kv_heads / hpc) * row_tiles(i);
        wide_rows |= sessions[i].q_rows * group > 8;
    }
    const uint32_t cluster = n_sessions <= kParamSessions ? cluster_size(ctx, keys, n_sessions, p, streams, wide_rows, hpc, rows_form) : 0u;
    *taken = cluster != 0;
    if (cluster == 0) return TT_OK;
    TTSessionTable &table = ctx->session_table;
    uint32_t ctas = 0;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        table.s[i] = sessions[i];
        table.item_prefix[i] = ctas;
        ctas += p->n_kv_heads / hpc * row_tiles(i) * cluster;
    }
    table.item_prefix[n_sessions] = ctas;
    table.n = n_sessions;
    const PassExtra<kPassSinkCluster> extra = {form.sink, form.window, cluster, p->out_row_stride_elements, nullptr};
    TTLaunchTimer timer(ctx, stream, TT_PROFILE_DECODE_PARTIAL);
    const cudaError_t e = launch_cluster(stream, ctas, extra, p, ctx->status, table, wide_rows, hpc);
    if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_sink launch");
    timer.stop();
    ctx->launches++;
    return TT_OK;
}

// First key of the union of the rows' windows behind the sinks, and the number of keys any row sees.
TT_API int tt_attn_sink_keys(uint32_t seq_len, uint32_t q_rows, uint32_t sink_tokens, uint32_t window,
                             uint32_t *out_window_start, uint32_t *out_keys) {
    if (q_rows == 0 || seq_len + 1ull < q_rows || seq_len > (uint32_t)INT32_MAX) return TT_ERR_INVALID_ARG;
    const uint32_t first_end = seq_len - (q_rows - 1);               // causal end of the first row
    uint32_t start = window != 0 && first_end > window ? first_end - window : 0u;
    if (start < sink_tokens) start = sink_tokens;
    if (start > seq_len) start = seq_len > sink_tokens ? seq_len : sink_tokens;
    if (out_window_start) *out_window_start = start;
    if (out_keys) *out_keys = (seq_len < sink_tokens ? seq_len : sink_tokens) + (seq_len > start ? seq_len - start : 0u);
    return TT_OK;
}

TT_API int tt_attn_decode_sink_window(tt_context *ctx, tt_stream stream, const tt_attn_session *sessions, uint32_t n_sessions,
                                      const tt_attn_batch_params *params, uint32_t sink_tokens, uint32_t window,
                                      uint32_t ring_capacity) {
    TT_ENTER(ctx);
    if (params == nullptr || (sessions == nullptr && n_sessions != 0))
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "sessions and params must not be null");
    if (n_sessions > ctx->max_sessions)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_sessions %u exceeds the context's max_sessions %u", n_sessions,
                            ctx->max_sessions);
    if (sink_tokens > (uint32_t)INT32_MAX) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "sink_tokens %u is too large", sink_tokens);
    if (ring_capacity != 0 && window == 0)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "a ring cache needs a window: without one every key stays visible");
    TTDecodeForm form;
    form.form = kPassSink;
    form.sink = sink_tokens;
    form.window = window == 0 || window > (uint32_t)INT32_MAX ? (uint32_t)INT32_MAX : window;
    TTDecodeSession *tmp = ctx->h_sessions_in;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        const tt_attn_session &s = sessions[i];
        TTDecodeSession &d = tmp[i];
        if (s.kv_start != 0) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: kv_start must be 0 (the window sets it)", i);
        uint32_t start = 0;
        if (tt_attn_sink_keys(s.seq_len, s.q_rows, sink_tokens, window, &start, nullptr) != TT_OK)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: seq_len %u cannot hold %u query rows", i, s.seq_len, s.q_rows);
        // the oldest key the first row sees must not have been overwritten by the last row's key
        if (ring_capacity != 0 && (uint64_t)ring_capacity < (uint64_t)window + s.q_rows - 1 &&
            (uint64_t)s.seq_len > (uint64_t)sink_tokens + ring_capacity)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: a ring of %u rows cannot hold a window of %u for %u rows", i,
                                ring_capacity, window, s.q_rows);
        d.q = s.q; d.out = s.out; d.k = s.k; d.v = s.v;
        d.seq_len = s.seq_len; d.q_rows = s.q_rows; d.kv_start = start;
        d.n_parts = 0; d.partial_base = 0; d.ring_capacity = ring_capacity; d.keep = nullptr; d.row_index = nullptr;
    }
    return tt_launch_decode(ctx, (cudaStream_t)stream, tmp, n_sessions, params, 0, nullptr, nullptr, nullptr, nullptr, nullptr, &form);
}
