// Decode attention that also adds every cached row's attention weight to a running statistic.
//
// A cache of a fixed number of rows keeps the rows that attention has used: the statistic of row j of a KV head is
// A[j] += sum over the session's query rows r and the head's query heads g of softmax(q_rg . K^T * scale)[j].
// A weight needs the maximum and the sum of its whole row, which exist only after all splits of the key range are
// done. Instead of reading K a second time, pass 1 (attn_pass1.cuh) leaves the raw scores behind (4 bytes per key and
// query head next to the 4 * head_dim bytes of K and V it reads per key and KV head; stored to stay in L2), and one
// launch behind it merges the output rows in its first CTAs and forms the weights from the scores in the others. The
// sums the weights divide by are those of the unrounded weights: the output divides by the sum of the ROUNDED ones its
// P.V product used, whose error (2^-9 with bf16 weights) the statistic, in 32 bits, would otherwise collect step after
// step. Every statistic is written by one thread in a fixed order, so results do not depend on the schedule.
//
// Bound: the bytes of K and V. 32 sessions of 1024 to 32768 keys, 16/2 heads of 256, bf16: 206 us a call, 5.4 TB/s, of
// which 15 us are the launch behind the pass; the same batch through plain decode 176 us. One session of 4096 keys 11 us.
#include "attn_merge.cuh"
#include "attn_pass1.cuh"

namespace {

constexpr uint32_t kAccThreads = 256;
constexpr uint32_t kAccPerThread = 4;                            // keys of one thread
constexpr uint32_t kAccKeys = kAccThreads * kAccPerThread;       // ... and of one CTA

struct AccSession {
    const float *scores;
    float *weights;              // row 0 of KV head 0
    uint32_t *positions;         // nullable
    void *out;
    uint32_t seq_len;            // keys the scores cover
    uint32_t total_len;          // keys of the whole session (>= seq_len when its rows are taken in several passes)
    uint32_t q_rows;
    uint32_t n_parts, partial_base;
    uint32_t fresh_begin;        // rows from here on start at zero (total_len: none)
    uint32_t end_position;
};

struct AccTable {
    uint32_t n, merge_ctas, merge_groups, merge_rows;
    uint32_t first_cta[kParamSessions];      // CTAs (behind the merge's) of the sessions before each one
    uint32_t first_row[kParamSessions];      // query rows of the sessions before each one
    AccSession s[kParamSessions];
};

struct AccParams {
    const float *part_o, *part_m, *part_l;
    const float *part_m2, *part_l2;
    uint32_t n_q_heads, n_kv_heads, row_pad, head_stride, out_row_stride;
    float scale_log2;
};

__device__ __forceinline__ uint32_t last_not_above(const uint32_t *first, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// grid = merge CTAs, then per session (key chunks x KV heads). In the latter a thread has four keys; the scores of its
// first eight rows are on their way while the rows' normalisers are merged from the parts' (max, sum), a warp per row.
template <typename T, int HD>
__global__ void __launch_bounds__(kAccThreads)
attn_accumulate_kernel(const __grid_constant__ AccTable table, AccParams p) {
    extern __shared__ float norm[];           // log2 of the softmax denominator of every packed row
    __shared__ typename RowMerge<HD>::Shared shared;
    pdl_launch_dependents();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (blockIdx.x < table.merge_ctas) {
        const uint32_t out_row = RowMerge<HD>::row(blockIdx.x, warp, table.merge_groups);
        const bool live = out_row < table.merge_rows;
        const uint32_t qrow = out_row / p.n_q_heads, head = out_row - qrow * p.n_q_heads;
        const uint32_t i = last_not_above(table.first_row, table.n, qrow);
        const AccSession &ses = table.s[i];
        const uint32_t w = qrow - table.first_row[i];
        RowMerge<HD> merge(warp, lane, table.merge_groups);
        pdl_wait();                           // pass 1 is done
        if (live)
            merge.walk(p.part_o, p.part_m, p.part_l, (size_t)ses.partial_base + w * p.n_q_heads + head, (size_t)ses.q_rows * p.n_q_heads, ses.n_parts);
        if (!merge.join(shared) || !live) return;
        merge.template store<T>(reinterpret_cast<T *>(ses.out) + (size_t)w * p.out_row_stride + (size_t)head * HD);
        return;
    }
    const uint32_t cta = blockIdx.x - table.merge_ctas, i = last_not_above(table.first_cta, table.n, cta);
    const AccSession &ses = table.s[i];
    const uint32_t local = cta - table.first_cta[i];
    const uint32_t kv_head = local % p.n_kv_heads, chunk = local / p.n_kv_heads;
    const uint32_t group = p.n_q_heads / p.n_kv_heads;
    const uint32_t rows = ses.q_rows * group, rows_padded = (rows + p.row_pad - 1) / p.row_pad * p.row_pad;
    const uint32_t rows_total = ses.q_rows * p.n_q_heads;
    const uint32_t seq_len = ses.seq_len, total_len = ses.total_len;
    const float *scores = ses.scores + (size_t)kv_head * seq_len * rows_padded;

    uint32_t key[kAccPerThread];
    float s[kAccPerThread][8], sum[kAccPerThread], old[kAccPerThread];
    auto load_rows = [&](uint32_t r0) {       // eight rows' scores of every key (the padding reaches a multiple of eight)
#pragma unroll
        for (uint32_t x = 0; x < kAccPerThread; ++x)
            if (key[x] < seq_len) {
                const float4 *row = reinterpret_cast<const float4 *>(scores + (size_t)key[x] * rows_padded + r0);
                const float4 a = row[0], b = row[1];
                s[x][0] = a.x; s[x][1] = a.y; s[x][2] = a.z; s[x][3] = a.w;
                s[x][4] = b.x; s[x][5] = b.y; s[x][6] = b.z; s[x][7] = b.w;
            }
    };
    float *weights = ses.weights + (size_t)kv_head * p.head_stride;
    pdl_wait();                               // pass 1 is done
#pragma unroll
    for (uint32_t x = 0; x < kAccPerThread; ++x) {
        key[x] = chunk * kAccKeys + x * kAccThreads + threadIdx.x;
        sum[x] = 0.f;
        old[x] = key[x] < min(total_len, ses.fresh_begin) ? weights[key[x]] : 0.f;
    }
    load_rows(0);
    for (uint32_t r = warp; r < rows; r += kAccThreads / 32) {
        const size_t base = (size_t)ses.partial_base + (r / group) * p.n_q_heads + kv_head * group + r % group;
        float m = -INFINITY, l = 0.f;
        for (uint32_t c = lane; c < ses.n_parts; c += 32) {
            const size_t at = base + (size_t)c * rows_total;
            const float m2 = p.part_m2[at], l2 = p.part_l2[at];
            const float m_new = fmaxf(m, m2);
            if (m_new != -INFINITY) l = l * exp2f(m - m_new) + l2 * exp2f(m2 - m_new);
            m = m_new;
        }
        float mx = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        l = mx != -INFINITY ? l * exp2f(m - mx) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) norm[r] = l > 0.f ? mx + log2f(l) : INFINITY;      // a row that sees nothing weighs nothing
    }
    __syncthreads();
    // query row w of q_rows sees keys below seq_len - (q_rows - 1 - w): the first `hidden` packed rows do not see a last key
    uint32_t hidden[kAccPerThread];
#pragma unroll
    for (uint32_t x = 0; x < kAccPerThread; ++x)
        hidden[x] = key[x] >= seq_len ? 0xffffffffu : key[x] + ses.q_rows > seq_len ? (key[x] + ses.q_rows - seq_len) * group : 0u;
    for (uint32_t r0 = 0; r0 < rows; r0 += 8) {
        if (r0 != 0) load_rows(r0);
#pragma unroll
        for (uint32_t y = 0; y < 8; ++y) {
            if (r0 + y >= rows) break;
            const float n = norm[r0 + y];
#pragma unroll
            for (uint32_t x = 0; x < kAccPerThread; ++x) {
                const float w = fast_exp2(fmaf(s[x][y], p.scale_log2, -n));      // 2^-22 relative
                sum[x] += r0 + y >= hidden[x] ? w : 0.f;
            }
        }
    }
#pragma unroll
    for (uint32_t x = 0; x < kAccPerThread; ++x) {
        if (key[x] >= total_len) continue;
        weights[key[x]] = old[x] + sum[x];
        if (key[x] >= ses.fresh_begin && ses.positions != nullptr)
            ses.positions[(size_t)kv_head * p.head_stride + key[x]] = ses.end_position - (total_len - key[x]);
    }
}

template <typename T>
cudaError_t launch_accumulate(cudaStream_t stream, uint32_t head_dim, uint32_t ctas, size_t smem, const AccTable &table, const AccParams &p) {
    switch (head_dim) {
        case 64: return tt_launch_pdl(attn_accumulate_kernel<T, 64>, dim3(ctas), dim3(kAccThreads), smem, stream, table, p);
        case 128: return tt_launch_pdl(attn_accumulate_kernel<T, 128>, dim3(ctas), dim3(kAccThreads), smem, stream, table, p);
        default: return tt_launch_pdl(attn_accumulate_kernel<T, 256>, dim3(ctas), dim3(kAccThreads), smem, stream, table, p);
    }
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

}  // namespace

cudaError_t tt_launch_pass1_scores(cudaStream_t stream, uint32_t n_items, const TTDecodeItem *items, const TTDecodeSession *sessions,
                                   const TTDecodeForm &form, const tt_attn_batch_params *p, uint32_t *status,
                                   const TTSessionTable &table, uint32_t table_keys, bool wide_rows, uint32_t hpc) {
    PassExtra<kPassScores> extra;
    extra.part_m2 = form.part_m2;
    extra.part_l2 = form.part_l2;
    if (p->io_dtype == TT_F16)
        return launch_partial_hd<__half>(stream, n_items, items, sessions, form.part_o, form.part_m, form.part_l, p, status,
                                         table, table_keys, wide_rows, hpc, extra);
    return launch_partial_hd<__nv_bfloat16>(stream, n_items, items, sessions, form.part_o, form.part_m, form.part_l, p, status,
                                            table, table_keys, wide_rows, hpc, extra);
}

TT_API int tt_attn_decode_accumulate(tt_context *ctx, tt_stream stream, const tt_attn_session *sessions,
                                     const tt_attn_weight_rows *weight_rows, uint32_t n_sessions,
                                     const tt_attn_batch_params *params, uint32_t head_stride) {
    TT_ENTER(ctx);
    if (params == nullptr || ((sessions == nullptr || weight_rows == nullptr) && n_sessions != 0))
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "sessions, weight rows and params must not be null");
    if (params->n_kv_heads == 0 || params->n_q_heads == 0 || params->n_q_heads % params->n_kv_heads != 0)
        return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_q_heads must be a multiple of n_kv_heads");
    if (params->n_q_heads > 96) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "n_q_heads exceeds 96");
    if (params->head_dim != 64 && params->head_dim != 128 && params->head_dim != 256)
        return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "decode attention supports head_dim 64/128/256, got %u", params->head_dim);
    if (!(params->scale > 0.f)) return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "accumulated weights need a positive scale");
    const uint32_t group = params->n_q_heads / params->n_kv_heads;
    for (uint32_t i = 0; i < n_sessions; ++i) {
        const tt_attn_session &s = sessions[i];
        const tt_attn_weight_rows &w = weight_rows[i];
        if (s.kv_start != 0) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: kv_start must be 0", i);
        if (s.q_rows == 0 || s.q_rows > 64) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: q_rows must be in 1..64", i);
        if (s.seq_len > (uint32_t)INT32_MAX || s.seq_len + 1 < s.q_rows)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: seq_len %u cannot hold %u query rows", i, s.seq_len, s.q_rows);
        if (s.q == nullptr || s.k == nullptr || s.v == nullptr || s.out == nullptr)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u has a null buffer", i);
        if (((uintptr_t)s.q | (uintptr_t)s.k | (uintptr_t)s.v | (uintptr_t)s.out) & 15)
            return tt_set_error(ctx, TT_ERR_UNSUPPORTED_SHAPE, "session %u: buffers must be 16-byte aligned", i);
        if (w.weights == nullptr) return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u has no weight row", i);
        if (((uintptr_t)w.weights | (uintptr_t)w.positions) & 3)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: weight and position rows must be 4-byte aligned", i);
        if (s.seq_len > head_stride)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: %u keys do not fit a weight row of %u", i, s.seq_len, head_stride);
        if (w.fresh_rows > s.seq_len)
            return tt_set_error(ctx, TT_ERR_INVALID_ARG, "session %u: %u fresh rows of %u", i, w.fresh_rows, s.seq_len);
    }
    // The scores of one pass share the workspace with its split partials: at most half of it. A batch that needs more
    // is taken in several passes, by sessions first, then by the query rows of one session.
    const size_t score_budget = ctx->workspace_bytes / 2 / 16 * 16;
    const uint32_t pass_sessions = ctx->max_sessions < kParamSessions ? ctx->max_sessions : kParamSessions;      // the context's tables hold no more
    struct Pass { uint32_t count, rows_of_first, pad; size_t bytes; };
    auto reserved = [](const Pass &pass) { return (pass.bytes + 255) / 256 * 256 + 16; };
    // the pass from query row `row_done` of session i on; no sessions: the scores of session i do not fit
    auto pass_from = [&](uint32_t i, uint32_t row_done) {
        Pass pass = {0, 0, 8, 0};
        // with 8-row padding when every session of the pass fits it, else with 16-row padding
        for (uint32_t pad = 8; pad <= 16; pad += 8) {
            bool wide_rows = false;
            pass.bytes = 0; pass.count = 0;
            for (uint32_t k = i; k < n_sessions && pass.count < pass_sessions; ++k) {
                const uint32_t all = sessions[k].q_rows - (k == i ? row_done : 0u);
                uint32_t rows = all;
                auto need = [&](uint32_t r) {
                    return (size_t)params->n_kv_heads * sessions[k].seq_len * ((r * group + pad - 1) / pad * pad) * sizeof(float);
                };
                if (pass.bytes + need(rows) > score_budget) {
                    if (pass.count != 0) break;
                    while (rows > 1 && need(rows) > score_budget) --rows;
                    if (need(rows) > score_budget) return pass;
                }
                pass.bytes += (need(rows) + 15) / 16 * 16;
                wide_rows |= rows * group > 8;
                if (pass.count == 0) pass.rows_of_first = rows;
                ++pass.count;
                if (rows != all) break;                  // a session cut by rows ends its pass
            }
            pass.pad = wide_rows ? 16u : 8u;             // what pass 1 pads these sessions to
            if (!wide_rows) break;
        }
        return pass;
    };
    // the rest of a cut session, or the sessions behind it
    auto advance = [&](const Pass &pass, uint32_t &i, uint32_t &row_done) {
        if (pass.count == 1 && row_done + pass.rows_of_first < sessions[i].q_rows) {
            row_done += pass.rows_of_first;
        } else {
            i += pass.count;
            row_done = 0;
        }
    };
    // A call whose later pass does not fit is refused before its first one has added to a statistic (a call of one pass is
    // refused by tt_launch_decode, before it launches).
    for (uint32_t i = 0, row_done = 0; i < n_sessions;) {
        const Pass pass = pass_from(i, row_done);
        if (pass.count == 0) return tt_set_error(ctx, TT_ERR_OOM, "the scores of session %u do not fit the context workspace", i);
        if (pass.count == n_sessions && pass.rows_of_first == sessions[0].q_rows) break;
        size_t room = ctx->workspace_bytes;
        room = room > reserved(pass) ? (room - reserved(pass)) / (params->head_dim + 4) * (params->head_dim + 2) : 0;
        for (uint32_t c = 0; c < pass.count; ++c) {
            const uint32_t skip = c == 0 ? row_done : 0u;
            ctx->h_rows[c] = c == 0 ? pass.rows_of_first : sessions[i + c].q_rows;
            ctx->h_keys[c] = sessions[i + c].seq_len - (sessions[i + c].q_rows - skip - ctx->h_rows[c]);
        }
        if (room == 0 || tt_attn_plan_splits(ctx->h_keys, ctx->h_rows, pass.count, params->head_dim, params->n_q_heads, params->n_kv_heads,
                                             (uint32_t)ctx->sm_count, room, nullptr, nullptr) != TT_OK)
            return tt_set_error(ctx, TT_ERR_OOM, "the partials of session %u do not fit the context workspace", i);
        advance(pass, i, row_done);
    }
    static thread_local AccTable table;
    uint32_t i = 0, row_done = 0;
    while (i < n_sessions) {
        const Pass pass = pass_from(i, row_done);
        const uint32_t count = pass.count, rows_of_first = pass.rows_of_first, pad = pass.pad;
        const size_t bytes = pass.bytes;
        TTDecodeSession *tmp = ctx->h_sessions_in;
        float *scores = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->partials) + (ctx->workspace_bytes / 16 * 16 - (bytes + 255) / 256 * 256));
        table.n = count;
        uint32_t blocks = 0, max_rows = 0, query_rows = 0;
        for (uint32_t c = 0; c < count; ++c) {
            const tt_attn_session &s = sessions[i + c];
            const uint32_t skip = c == 0 ? row_done : 0u, rows = c == 0 ? rows_of_first : s.q_rows;
            TTDecodeSession &d = tmp[c];
            d.q = reinterpret_cast<const unsigned char *>(s.q) + (size_t)skip * params->q_row_stride_elements * 2;
            d.out = s.out;                   // pass 1 leaves it alone
            d.k = s.k; d.v = s.v;
            d.seq_len = s.seq_len - (s.q_rows - skip - rows); d.q_rows = rows; d.kv_start = 0;
            d.n_parts = 0; d.partial_base = 0; d.ring_capacity = 0; d.keep = nullptr; d.scores = scores;
            AccSession &a = table.s[c];
            a.scores = scores;
            a.weights = weight_rows[i + c].weights; a.positions = weight_rows[i + c].positions;
            a.seq_len = d.seq_len; a.total_len = s.seq_len; a.q_rows = rows;
            a.fresh_begin = skip == 0 ? s.seq_len - weight_rows[i + c].fresh_rows : s.seq_len;
            a.end_position = weight_rows[i + c].end_position;
            a.out = reinterpret_cast<unsigned char *>(s.out) + (size_t)skip * params->out_row_stride_elements * 2;
            table.first_cta[c] = blocks;
            table.first_row[c] = query_rows;
            query_rows += rows;
            blocks += ceil_div(s.seq_len, kAccKeys) * params->n_kv_heads;
            const uint32_t padded = (rows * group + pad - 1) / pad * pad;
            scores += ((size_t)params->n_kv_heads * d.seq_len * padded + 3) / 4 * 4;
            if (rows * group > max_rows) max_rows = rows * group;
        }
        TTDecodeForm form;
        form.form = kPassScores;
        form.partials_only = true;
        form.reserved_bytes = reserved(pass);
        int rc = tt_launch_decode(ctx, (cudaStream_t)stream, tmp, count, params, 0, nullptr, nullptr, nullptr, nullptr, nullptr, &form);
        if (rc != TT_OK) return rc;
        uint32_t max_parts = 0;
        for (uint32_t c = 0; c < count; ++c) {
            table.s[c].n_parts = ctx->h_sessions[c].n_parts;
            table.s[c].partial_base = ctx->h_sessions[c].partial_base;
            if (ctx->h_sessions[c].n_parts > max_parts) max_parts = ctx->h_sessions[c].n_parts;
        }
        table.merge_rows = query_rows * params->n_q_heads;
        table.merge_groups = merge_groups(table.merge_rows, max_parts, params->head_dim, (uint32_t)ctx->sm_count, &table.merge_ctas);
        AccParams p;
        p.part_o = form.part_o; p.part_m = form.part_m; p.part_l = form.part_l; p.part_m2 = form.part_m2; p.part_l2 = form.part_l2;
        p.n_q_heads = params->n_q_heads; p.n_kv_heads = params->n_kv_heads; p.row_pad = pad; p.head_stride = head_stride;
        p.out_row_stride = params->out_row_stride_elements; p.scale_log2 = params->scale * kLog2e;
        const uint32_t ctas = table.merge_ctas + blocks;
        const size_t smem = max_rows * sizeof(float);
        const cudaError_t e = params->io_dtype == TT_F16 ? launch_accumulate<__half>((cudaStream_t)stream, params->head_dim, ctas, smem, table, p)
                                                         : launch_accumulate<__nv_bfloat16>((cudaStream_t)stream, params->head_dim, ctas, smem, table, p);
        if (e != cudaSuccess) return tt_check_cuda(ctx, e, "attn_accumulate launch");
        ctx->launches++;
        advance(pass, i, row_done);
    }
    return TT_OK;
}
