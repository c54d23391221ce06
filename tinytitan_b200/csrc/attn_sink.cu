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
// the visible rows. With one row every fetched key is visible and no score is masked.
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
