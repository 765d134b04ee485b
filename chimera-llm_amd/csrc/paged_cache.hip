// Norms of query and key heads with the position rotation in the same pass (lcmhip_head_norm_rope), and the same on the way into
// the pages of a cache (lcmhip_paged_append).
//
// One kernel.  A head of D values is held by D / 8 lanes, 8 consecutive values each (one 16-byte load in bf16, two in fp32):
//     rms       y = x / sqrt(mean(x^2) + eps) * w
//     standard  y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * w + b
//     rotation  (y_i, y_j) -> (y_i cos - y_j sin, y_i sin + y_j cos), j = i + 1 or i + rotary_dim / 2
// in fp32, rounded once when it is stored.  The sums run over the D / 8 lanes of a head; the partner of a pair (i, i + 1) is
// in the same lane, that of (i, i + rotary_dim / 2) rotary_dim / 16 lanes away.
#include "paged.h"

namespace lcmhip {

struct HeadArgs {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    void *q_out, *k_out;                                       // k_out: plain rows (head_norm_rope only)
    int64_t qo_row, qo_head, ko_row, ko_head;
    int64_t rows;
    int nq, nk, nv;                                            // heads of each kind in a row (0: none)
    lcmhip_head_norm norm;
    lcmhip_rotary rot;                                         // rotary_dim 0: none
    const int32_t* positions;
    // append
    void *k_pages, *v_pages;
    PageTable table;
    const int32_t *seq_lens, *q_starts;
    int n_seqs, max_keys;
};

// Eight values as they lie in memory.
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16_t> { uint4 x; };
template <>
struct Raw8<float> { float4 x, y; };

// HPT heads for each lane group; SLOTS * HPT consecutive heads (query heads, key heads, value heads of row 0, of row 1, ..)
// for each workgroup.  All loads of a lane group's heads are in flight before the first is worked on.
template <typename T, int D, bool APPEND, int HPT>
__global__ __launch_bounds__(256) void k_head_rows(HeadArgs a) {
    constexpr int LPH = D / 8, SLOTS = 256 / LPH;
    const int nh = a.nq + a.nk + a.nv;
    const int64_t base = (int64_t)blockIdx.x * (SLOTS * HPT);
    const int64_t row0 = base / nh;
    const int rem0 = (int)(base - row0 * nh);
    const int slot = threadIdx.x / LPH, sub = threadIdx.x % LPH, i0 = sub * 8;
    int seq0 = 0;
    if (APPEND && a.q_starts) seq0 = wave_count_le(a.q_starts + 1, a.n_seqs, row0);

    Raw8<T> raw[HPT];
    T* dst[HPT];
    int kinds[HPT], poss[HPT];
#pragma unroll
    for (int it = 0; it < HPT; ++it) {
        const unsigned u = (unsigned)rem0 + slot + it * SLOTS;
        const int64_t row = row0 + u / (unsigned)nh;
        int h = (int)(u % (unsigned)nh);
        bool live = row < a.rows;
        const int kind = h < a.nq ? 0 : (h < a.nq + a.nk ? 1 : 2);
        if (kind >= 1) h -= a.nq;
        if (kind == 2) h -= a.nk;
        const T* src = kind == 0 ? reinterpret_cast<const T*>(a.q) + row * a.q_row + h * a.q_head
                                 : (kind == 1 ? reinterpret_cast<const T*>(a.k) + row * a.k_row + h * a.k_head
                                              : reinterpret_cast<const T*>(a.v) + row * a.v_row + h * a.v_head);
        raw[it] = Raw8<T>{};
        if (live) raw[it] = *reinterpret_cast<const Raw8<T>*>(src + i0);
        int pos = 0;
        T* to = nullptr;
        if (APPEND) {
            int c = -1, seq = seq0;
            if (live) {
                if (a.q_starts) {
                    while (seq < a.n_seqs && a.q_starts[seq + 1] <= row) ++seq;   // a few rows past row0: almost never a step
                } else {
                    seq = (int)row;
                }
                if (seq < a.n_seqs) {
                    int64_t r0, r1;
                    seq_rows(a.q_starts, seq, a.rows, r0, r1);
                    const int len = max(0, min(a.seq_lens[seq], a.max_keys));
                    if (row >= r0) c = (int)max((int64_t)-1, len - (r1 - row));
                }
            }
            pos = a.positions && live ? a.positions[row] : c;
            live = c >= 0 && pos >= 0;
            if (live && kind >= 1) {
                const int page = a.table.page(seq, c);
                if (page >= 0) {
                    const int off = c & ((1 << a.table.page_shift) - 1);
                    T* pool = reinterpret_cast<T*>(kind == 1 ? a.k_pages : a.v_pages);
                    to = pool + ((((size_t)page * a.nk + h) << a.table.page_shift) + off) * D + i0;
                }
            } else if (live) {
                to = reinterpret_cast<T*>(a.q_out) + row * a.qo_row + h * a.qo_head + i0;
            }
        } else if (live) {
            pos = a.positions ? a.positions[row] : 0;
            if (pos >= 0)
                to = kind == 0 ? reinterpret_cast<T*>(a.q_out) + row * a.qo_row + h * a.qo_head + i0
                               : reinterpret_cast<T*>(a.k_out) + row * a.ko_row + h * a.ko_head + i0;
        }
        dst[it] = to;
        kinds[it] = kind;
        poss[it] = pos;
    }
#pragma unroll
    for (int it = 0; it < HPT; ++it) {
        if (kinds[it] == 2) {                              // values go as they are
            if (dst[it]) *reinterpret_cast<Raw8<T>*>(dst[it]) = raw[it];
            continue;
        }
        float x[8];
        load8<T>(reinterpret_cast<const T*>(&raw[it]), x);
        if (a.norm.kind != LCMHIP_NORM_NONE) {
            if (a.norm.kind != LCMHIP_NORM_RMS) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += x[j];
#pragma unroll
                for (int off = LPH / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] -= s * (1.f / D);
            }
            float s2 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s2 += x[j] * x[j];
#pragma unroll
            for (int off = LPH / 2; off > 0; off >>= 1) s2 += __shfl_xor(s2, off, 64);
            const float r = 1.f / sqrtf(s2 * (1.f / D) + a.norm.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= r;
            const void* w = kinds[it] == 0 ? a.norm.q_weight : a.norm.k_weight;
            const void* b = kinds[it] == 0 ? a.norm.q_bias : a.norm.k_bias;
            if (w) {
                float wv[8];
                load8<T>(reinterpret_cast<const T*>(w) + i0, wv);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= wv[j];
            }
            if (b) {
                float bv[8];
                load8<T>(reinterpret_cast<const T*>(b) + i0, bv);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] += bv[j];
            }
        }
        if (a.rot.rotary_dim > 0) {
            const int half = a.rot.rotary_dim >> 1, pos = poss[it];
            const bool known = pos < a.rot.n_positions;
            const size_t trow = (size_t)(known ? max(pos, 0) : 0) * half;
            if (a.rot.style == LCMHIP_ROTARY_PAIRS) {
                if (i0 < a.rot.rotary_dim) {
                    const float4 cs = *reinterpret_cast<const float4*>(a.rot.cos + trow + i0 / 2);
                    const float4 sn = *reinterpret_cast<const float4*>(a.rot.sin + trow + i0 / 2);
                    rope_rotate(x[0], x[1], cs.x, sn.x);
                    rope_rotate(x[2], x[3], cs.y, sn.y);
                    rope_rotate(x[4], x[5], cs.z, sn.z);
                    rope_rotate(x[6], x[7], cs.w, sn.w);
                }
            } else {
                const bool first = i0 < half;
                const int lane = threadIdx.x & 63;
                const int partner = i0 < a.rot.rotary_dim ? lane + (first ? half / 8 : -(half / 8)) : lane;
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = __shfl(x[j], partner, 64);
                if (i0 < a.rot.rotary_dim) {
                    float cs[8], sn[8];
                    load8<float>(a.rot.cos + trow + (first ? i0 : i0 - half), cs);
                    load8<float>(a.rot.sin + trow + (first ? i0 : i0 - half), sn);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = first ? x[j] * cs[j] - y[j] * sn[j] : x[j] * cs[j] + y[j] * sn[j];
                }
            }
            if (!known) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_nanf("");
            }
        }
        if (dst[it]) store8<T>(dst[it], x);
    }
}

template <typename T, int D, bool APPEND>
static int launch_head_rows_t(const HeadArgs& a, hipStream_t st) {
    constexpr int SLOTS = 256 / (D / 8);
    const int64_t heads = a.rows * (a.nq + a.nk + a.nv);
    if (heads == 0) return LCMHIP_OK;
    // four heads a lane group once that still fills the chip's 256 CUs with eight workgroups each, else one
    const int hpt = heads >= (int64_t)SLOTS * 4 * 2048 ? 4 : 1;
    const int64_t blocks = (heads + SLOTS * hpt - 1) / (SLOTS * hpt);
    LCM_REQUIRE(blocks <= INT32_MAX, "head rows: too many rows");
    if (hpt == 4) hipLaunchKernelGGL((k_head_rows<T, D, APPEND, 4>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_head_rows<T, D, APPEND, 1>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    LCM_HIP_CHECK(hipGetLastError());
    return LCMHIP_OK;
}

static int launch_head_rows(const HeadArgs& a, int head_dim, int dtype, bool append, hipStream_t st) {
    if (dtype == LCMHIP_BF16) {
        if (head_dim == 64) return append ? launch_head_rows_t<bf16_t, 64, true>(a, st) : launch_head_rows_t<bf16_t, 64, false>(a, st);
        return append ? launch_head_rows_t<bf16_t, 128, true>(a, st) : launch_head_rows_t<bf16_t, 128, false>(a, st);
    }
    if (head_dim == 64) return append ? launch_head_rows_t<float, 64, true>(a, st) : launch_head_rows_t<float, 64, false>(a, st);
    return append ? launch_head_rows_t<float, 128, true>(a, st) : launch_head_rows_t<float, 128, false>(a, st);
}

// Takes over norm and rotary (NULL: none) after checking them.
static int take_transform(HeadArgs& a, const lcmhip_head_norm* norm, const lcmhip_rotary* rotary, int head_dim, bool with_q, bool with_k) {
    a.norm.kind = LCMHIP_NORM_NONE;
    if (norm) {
        const bool known = norm->kind == LCMHIP_NORM_NONE || norm->kind == LCMHIP_NORM_LAYERNORM || norm->kind == LCMHIP_NORM_RMS ||
                           norm->kind == LCMHIP_NORM_FP32 || norm->kind == LCMHIP_NORM_UNIT;
        LCM_REQUIRE(known, "head norm: unknown norm kind");
        const bool weights = norm->kind != LCMHIP_NORM_NONE && norm->kind != LCMHIP_NORM_UNIT;
        LCM_REQUIRE(!weights || ((!with_q || norm->q_weight) && (!with_k || norm->k_weight)), "head norm: this kind needs weights");
        LCM_REQUIRE(weights || !(norm->q_weight || norm->k_weight), "head norm: this kind has no weights");
        LCM_REQUIRE(norm->kind == LCMHIP_NORM_LAYERNORM || !(norm->q_bias || norm->k_bias), "head norm: this kind has no bias");
        LCM_REQUIRE(((uintptr_t)norm->q_weight | (uintptr_t)norm->k_weight | (uintptr_t)norm->q_bias | (uintptr_t)norm->k_bias) % 16 == 0,
                    "head norm: weights must be 16-byte aligned");
        LCM_REQUIRE(norm->eps >= 0.f, "head norm: eps must not be negative");
        a.norm = *norm;
    }
    a.rot.rotary_dim = 0;
    if (rotary) {
        LCM_REQUIRE(rotary->cos && rotary->sin, "rotary: null table");
        LCM_REQUIRE(rotary->rotary_dim >= 16 && rotary->rotary_dim <= head_dim && rotary->rotary_dim % 16 == 0,
                    "rotary: rotary_dim must be a multiple of 16 up to head_dim");
        LCM_REQUIRE(rotary->style == LCMHIP_ROTARY_PAIRS || rotary->style == LCMHIP_ROTARY_HALVES, "rotary: unknown style");
        LCM_REQUIRE(rotary->n_positions >= 1, "rotary: empty table");
        LCM_REQUIRE(((uintptr_t)rotary->cos | (uintptr_t)rotary->sin) % 16 == 0, "rotary: tables must be 16-byte aligned");
        a.rot = *rotary;
    }
    return LCMHIP_OK;
}

}  // namespace lcmhip

using namespace lcmhip;

extern "C" {

int lcmhip_head_norm_rope(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                          void* q_out, int64_t q_out_row, int64_t q_out_head, void* k_out, int64_t k_out_row, int64_t k_out_head,
                          int64_t rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const lcmhip_head_norm* norm,
                          const lcmhip_rotary* rotary, const int32_t* positions, int32_t dtype, void* stream) {
    LCM_REQUIRE(q || k, "head_norm_rope: neither queries nor keys");
    LCM_REQUIRE(!q == !q_out && !k == !k_out, "head_norm_rope: an input without its output");
    LCM_REQUIRE(dtype == LCMHIP_F32 || dtype == LCMHIP_BF16, "head_norm_rope: unknown dtype");
    LCM_REQUIRE(head_dim == 64 || head_dim == 128, "head_norm_rope: head_dim must be 64 or 128");
    LCM_REQUIRE(rows >= 0 && rows <= (1 << 30), "head_norm_rope: rows out of range");
    LCM_REQUIRE((!q || (n_heads >= 1 && n_heads <= 65535)) && (!k || (n_kv_heads >= 1 && n_kv_heads <= 65535)),
                "head_norm_rope: head count out of range");
    LCM_REQUIRE(!rotary || positions, "head_norm_rope: a rotation needs positions");
    LCM_TRY(check_rows(q, q_row, q_head, dtype, "head_norm_rope: q"));
    LCM_TRY(check_rows(k, k_row, k_head, dtype, "head_norm_rope: k"));
    LCM_TRY(check_rows(q_out, q_out_row, q_out_head, dtype, "head_norm_rope: q_out"));
    LCM_TRY(check_rows(k_out, k_out_row, k_out_head, dtype, "head_norm_rope: k_out"));
    LCM_REQUIRE(q != q_out || !q || (q_row == q_out_row && q_head == q_out_head), "head_norm_rope: in place needs equal strides");
    LCM_REQUIRE(k != k_out || !k || (k_row == k_out_row && k_head == k_out_head), "head_norm_rope: in place needs equal strides");
    HeadArgs a{};
    LCM_TRY(take_transform(a, norm, rotary, head_dim, q != nullptr, k != nullptr));
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.k = k; a.k_row = k_row; a.k_head = k_head;
    a.q_out = q_out; a.qo_row = q_out_row; a.qo_head = q_out_head;
    a.k_out = k_out; a.ko_row = k_out_row; a.ko_head = k_out_head;
    a.rows = rows; a.nq = q ? n_heads : 0; a.nk = k ? n_kv_heads : 0;
    a.positions = rotary ? positions : nullptr;
    return launch_head_rows(a, head_dim, dtype, false, static_cast<hipStream_t>(stream));
}

int lcmhip_paged_append(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const void* k, int64_t k_row, int64_t k_head,
                        const void* v, int64_t v_row, int64_t v_head, const void* q, int64_t q_row, int64_t q_head, void* q_out,
                        int64_t rows, int32_t n_heads, const lcmhip_head_norm* norm, const lcmhip_rotary* rotary,
                        const int32_t* positions, void* stream) {
    LCM_TRY(check_pages(pages));
    LCM_TRY(check_batch(pages, batch, rows));
    LCM_REQUIRE(k && v, "paged_append: null argument");
    LCM_REQUIRE(!q == !q_out, "paged_append: q and q_out come together");
    LCM_REQUIRE(!q || (n_heads >= 1 && n_heads <= 65535), "paged_append: head count out of range");
    LCM_TRY(check_rows(k, k_row, k_head, pages->dtype, "paged_append: k"));
    LCM_TRY(check_rows(v, v_row, v_head, pages->dtype, "paged_append: v"));
    LCM_TRY(check_rows(q, q_row, q_head, pages->dtype, "paged_append: q"));
    LCM_TRY(check_rows(q_out, 0, 0, pages->dtype, "paged_append: q_out"));
    HeadArgs a{};
    LCM_TRY(take_transform(a, norm, rotary, pages->head_dim, q != nullptr, true));
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.k = k; a.k_row = k_row; a.k_head = k_head;
    a.v = v; a.v_row = v_row; a.v_head = v_head;
    a.q_out = q_out; a.qo_head = pages->head_dim; a.qo_row = (int64_t)n_heads * pages->head_dim;
    a.rows = rows; a.nq = q ? n_heads : 0; a.nk = a.nv = pages->n_kv_heads;
    a.positions = positions;
    a.k_pages = pages->k; a.v_pages = pages->v;
    a.table = PageTable{batch->page_table, batch->max_pages, page_shift_of(pages), (uint32_t)pages->n_pages};
    a.seq_lens = batch->seq_lens; a.q_starts = batch->q_starts; a.n_seqs = batch->n_seqs; a.max_keys = batch->max_keys;
    return launch_head_rows(a, pages->head_dim, pages->dtype, true, static_cast<hipStream_t>(stream));
}

}  // extern "C"
