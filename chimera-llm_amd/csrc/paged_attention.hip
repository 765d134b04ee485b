// Attention of a ragged batch over the pages of its sequences, with or without prefixes that groups of sequences share.
//
// One wave for each (row, query head); lane = (key slot ks = lane / 4, dim group dg = lane % 4) walks the keys ks, ks + 16, ..
// with an online softmax (running maximum, sum and D / 4 accumulators a lane); the 16 slots are merged with shuffles at the
// end.  Sixteen keys of one step lie in one page, whose id is read once for the step.
#include "paged.h"

namespace lcmhip {

struct PagedArgs {
    const void* q; int64_t q_row, q_head;
    void* out;
    const void *kp, *vp;
    PageTable table, prefix_table;
    const int32_t *seq_lens, *q_starts, *prefix_lens, *group_starts;
    int n_seqs, n_groups, max_keys, prefix_max_keys;
    int64_t rows;
    int hq, hk, causal;
    float scale_log2;          // scale * log2(e).  It multiplies differences of dot products only: a product that fits fp32
                               // may leave it when multiplied by log2(e), and far from zero its rounding is no small number
};

template <typename T, int D>
__global__ __launch_bounds__(64) void k_paged_rows(PagedArgs a) {
    constexpr int P = D / 32;                       // 8-value pieces of a lane
    const int64_t row = blockIdx.x / a.hq;
    const int head = blockIdx.x % a.hq, hk = head / (a.hq / a.hk);
    const int lane = threadIdx.x, ks = lane >> 2, dg = lane & 3;
    const int seq = a.q_starts ? wave_count_le(a.q_starts + 1, a.n_seqs, row) : (int)row;
    if (seq >= a.n_seqs) return;
    int64_t r0, r1;
    seq_rows(a.q_starts, seq, a.rows, r0, r1);
    if (row < r0) return;
    const int len = max(0, min(a.seq_lens[seq], a.max_keys));
    const int keys = (int)max((int64_t)0, a.causal ? len - (r1 - row) + 1 : (int64_t)len);
    int group = a.n_groups, prefix = 0;
    if (a.n_groups > 0) {
        group = wave_count_le(a.group_starts + 1, a.n_groups, seq);
        if (group < a.n_groups && a.group_starts[group] <= seq) prefix = max(0, min(a.prefix_lens[group], a.prefix_max_keys));
    }
    const int col = dg * 8;
    float qv[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        load8<T>(reinterpret_cast<const T*>(a.q) + row * a.q_row + head * a.q_head + col + 32 * i, qv[i]);
    }
    float m = -INFINITY, l = 0.f, acc[P][8] = {};
    bool seen = false;
    auto walk = [&](const PageTable& table, int which, int count) {
        for (int k0 = 0; k0 < count; k0 += 16) {
            const int page = table.page(which, k0);
            if (page < 0) continue;
            const int key = k0 + ks;
            if (key >= count) continue;             // the 4 lanes of a slot agree
            const size_t at = ((((size_t)page * a.hk + hk) << table.page_shift) + (key & ((1 << table.page_shift) - 1))) * D + col;
            float s = 0.f, vv[P][8];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                float kv[8];
                load8<T>(reinterpret_cast<const T*>(a.kp) + at + 32 * i, kv);
                load8<T>(reinterpret_cast<const T*>(a.vp) + at + 32 * i, vv[i]);
#pragma unroll
                for (int t = 0; t < 8; ++t) s += kv[t] * qv[i][t];
            }
            s += __shfl_xor(s, 1, 64);
            s += __shfl_xor(s, 2, 64);
            seen = true;
            const float mn = fmaxf(m, s), ref = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2f((m - ref) * a.scale_log2), p = exp2f((s - ref) * a.scale_log2);
            l = l * alpha + p;
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int t = 0; t < 8; ++t) acc[i][t] = acc[i][t] * alpha + p * vv[i][t];
            m = mn;
        }
    };
    if (prefix > 0) walk(a.prefix_table, group, prefix);
    walk(a.table, seq, keys);
    float M = m;
#pragma unroll
    for (int off = 4; off <= 32; off <<= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    const float f = seen ? exp2f((m - (M == -INFINITY ? 0.f : M)) * a.scale_log2) : 0.f;
    float L = l * f;
#pragma unroll
    for (int off = 4; off <= 32; off <<= 1) L += __shfl_xor(L, off, 64);
    const bool any = __any(seen);                  // a row that sees no key gives zeros; 0 / 0 elsewhere is the formula's
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            float x = acc[i][t] * f;
#pragma unroll
            for (int off = 4; off <= 32; off <<= 1) x += __shfl_xor(x, off, 64);
            acc[i][t] = any ? x / L : 0.f;
        }
        if (ks == 0) store8<T>(reinterpret_cast<T*>(a.out) + ((size_t)row * a.hq + head) * D + col + 32 * i, acc[i]);
    }
}

static int check_prefix(const lcmhip_kv_pages* pages, const lcmhip_shared_prefix* prefix) {
    LCM_REQUIRE(prefix && prefix->page_table && prefix->lens && prefix->group_starts, "shared prefix: null argument");
    LCM_REQUIRE(prefix->n_groups >= 1 && prefix->n_groups <= (1 << 24), "shared prefix: n_groups out of range");
    LCM_REQUIRE(prefix->max_pages >= 1, "shared prefix: max_pages must be positive");
    LCM_REQUIRE(prefix->max_keys >= 1 && prefix->max_keys <= (int64_t)prefix->max_pages * pages->page_size,
                "shared prefix: max_keys must be in [1, max_pages * page_size]");
    return LCMHIP_OK;
}

static int check_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, int64_t rows, int n_heads) {
    LCM_TRY(check_pages(pages));
    LCM_TRY(check_batch(pages, batch, rows));
    LCM_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_heads % pages->n_kv_heads == 0,
                "paged attention: n_heads must be a multiple of n_kv_heads");
    LCM_REQUIRE(rows * n_heads <= INT32_MAX, "paged attention: too many rows");
    return LCMHIP_OK;
}

static int paged_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const lcmhip_shared_prefix* prefix,
                           const void* q, int64_t q_row, int64_t q_head, void* out, int64_t rows, int n_heads, float scale,
                           int causal, void* ws, size_t ws_bytes, hipStream_t st) {
    LCM_TRY(check_attention(pages, batch, rows, n_heads));
    if (prefix) LCM_TRY(check_prefix(pages, prefix));
    LCM_REQUIRE(q && out, "paged attention: null argument");
    LCM_REQUIRE(scale > 0.f && scale < INFINITY, "paged attention: scale must be positive and finite");
    LCM_TRY(check_rows(q, q_row, q_head, pages->dtype, "paged attention: q"));
    LCM_TRY(check_rows(out, 0, 0, pages->dtype, "paged attention: out"));
    if (rows == 0 || batch->n_seqs == 0) return LCMHIP_OK;
    PagedArgs a{};
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.out = out; a.kp = pages->k; a.vp = pages->v;
    a.table = PageTable{batch->page_table, batch->max_pages, page_shift_of(pages), pages->n_pages};
    a.seq_lens = batch->seq_lens; a.q_starts = batch->q_starts; a.n_seqs = batch->n_seqs; a.max_keys = batch->max_keys;
    if (prefix) {
        a.prefix_table = PageTable{prefix->page_table, prefix->max_pages, page_shift_of(pages), pages->n_pages};
        a.prefix_lens = prefix->lens; a.group_starts = prefix->group_starts;
        a.n_groups = prefix->n_groups; a.prefix_max_keys = prefix->max_keys;
    }
    a.rows = rows; a.hq = n_heads; a.hk = pages->n_kv_heads; a.causal = causal;
    a.scale_log2 = scale * 1.4426950408889634f;
    const dim3 grid((unsigned)(rows * n_heads)), block(64);
    if (pages->dtype == LCMHIP_BF16) {
        if (pages->head_dim == 64) hipLaunchKernelGGL((k_paged_rows<bf16_t, 64>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_paged_rows<bf16_t, 128>), grid, block, 0, st, a);
    } else {
        if (pages->head_dim == 64) hipLaunchKernelGGL((k_paged_rows<float, 64>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((k_paged_rows<float, 128>), grid, block, 0, st, a);
    }
    LCM_HIP_CHECK(hipGetLastError());
    return LCMHIP_OK;
}

}  // namespace lcmhip

using namespace lcmhip;

extern "C" {

int lcmhip_paged_attention_workspace(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, int64_t rows, int32_t n_heads,
                                     size_t* bytes) {
    LCM_REQUIRE(bytes, "paged_attention_workspace: null argument");
    LCM_TRY(check_attention(pages, batch, rows, n_heads));
    *bytes = 0;
    return LCMHIP_OK;
}

int lcmhip_paged_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const void* q, int64_t q_row, int64_t q_head,
                           void* out, int64_t rows, int32_t n_heads, float scale, int32_t causal, void* workspace,
                           size_t workspace_bytes, void* stream) {
    return paged_attention(pages, batch, nullptr, q, q_row, q_head, out, rows, n_heads, scale, causal, workspace, workspace_bytes,
                           static_cast<hipStream_t>(stream));
}

int lcmhip_shared_prefix_attention_workspace(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch,
                                             const lcmhip_shared_prefix* prefix, int64_t rows, int32_t n_heads, size_t* bytes) {
    LCM_REQUIRE(bytes, "shared_prefix_attention_workspace: null argument");
    LCM_TRY(check_attention(pages, batch, rows, n_heads));
    LCM_TRY(check_prefix(pages, prefix));
    *bytes = 0;
    return LCMHIP_OK;
}

int lcmhip_shared_prefix_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const lcmhip_shared_prefix* prefix,
                                   const void* q, int64_t q_row, int64_t q_head, void* out, int64_t rows, int32_t n_heads, float scale,
                                   int32_t causal, void* workspace, size_t workspace_bytes, void* stream) {
    LCM_REQUIRE(prefix, "shared_prefix_attention: null argument");
    return paged_attention(pages, batch, prefix, q, q_row, q_head, out, rows, n_heads, scale, causal, workspace, workspace_bytes,
                           static_cast<hipStream_t>(stream));
}

}  // extern "C"
