// Norms of query and key heads with the position rotation in the same pass (lcmhip_head_norm_rope), and the same on the way into
// the pages of a cache (lcmhip_paged_append).
//
// One kernel.  A head of D values is held by D / 8 lanes, 8 consecutive values each (one 16-byte load in bf16, two in fp32):
//     rms       y = x / sqrt(mean(x^2) + eps) * w
//     standard  y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * w + b
//     rotation  (y_i, y_j) -> (y_i cos - y_j sin, y_i sin + y_j cos), j = i + 1 or i + rotary_dim / 2
// in fp32, rounded once when it is stored.  The sums run over the D / 8 lanes of a head; the partner of a pair (i, i + 1) is
// in the same lane, that of (i, i + rotary_dim / 2) rotary_dim / 16 lanes away.
//
// Bound by bytes read and written, each once: 16384 rows of 32 + 8 heads of 128, bf16, in 64 us a call and 59 in the kernel (5.8 TB/s; a
// large copy reaches 5.0), 13 thousand rows of 32 + 8 + 8 heads appended behind ragged histories in 65 and 56 us (5.9 TB/s); 64 rows in
// 3.6 us, a launch.  A head at a time, with its angles and its place looked up for each, took 96 and 127 us a call: 220 vector
// operations a kilobyte.
#include <algorithm>

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

// Eight values as they lie in memory, read past the caches: nobody reads them again (append of 13 thousand rows, calls: 67 -> 60 us on
// one card).
// What is written stays in reach of the attention behind.
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16_t> {
    nv_u4 x;
    __device__ __forceinline__ void load(const bf16_t* p) { x = __builtin_nontemporal_load(reinterpret_cast<const nv_u4*>(p)); }
};
template <>
struct Raw8<float> {
    nv_u4 x, y;
    __device__ __forceinline__ void load(const float* p) {
        x = __builtin_nontemporal_load(reinterpret_cast<const nv_u4*>(p));
        y = __builtin_nontemporal_load(reinterpret_cast<const nv_u4*>(p) + 1);
    }
};

// Value of another lane of the same 16, as an operand modifier of a vector operation (no LDS).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over the 8 or 16 lanes of a head: neighbours, pairs, mirrored halves (0xB1 / 0x4E: lane ^ 1 / ^ 2, 0x141: mirrored in 8
// lanes, 0x140: mirrored in 16).
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    if (LPH == 16) v += dpp<0x140>(v);
    return v;
}

// A lane group keeps one row -- its place in the cache and its angles are looked up once -- and takes every (1 << head_shift)-th
// head of the workgroup's share of heads, CHUNK of them with their loads in flight together.
template <typename T, int D, bool APPEND, int CHUNK>
__global__ __launch_bounds__(256) void k_head_rows(HeadArgs a, int head_shift, int heads_per_block) {
    constexpr int LPH = D / 8, SLOTS = 256 / LPH;
    const int slot = threadIdx.x / LPH, i0 = (threadIdx.x % LPH) * 8;
    const int hs = 1 << head_shift, nh = a.nq + a.nk + a.nv;
    const int64_t block_row = (int64_t)blockIdx.x * (SLOTS >> head_shift);
    const int64_t r = block_row + (slot >> head_shift);
    bool live = r < a.rows;
    const int row = live ? (int)r : 0;
    int h = blockIdx.y * heads_per_block + (slot & (hs - 1));
    const int h1 = min(nh, (int)(blockIdx.y + 1) * heads_per_block);

    int pos = 0, page = -1;
    size_t in_pool = 0;                                    // of key head 0 at this row's place
    if (APPEND) {
        int seq = row;
        if (a.q_starts) {
            seq = wave_count_le(a.q_starts + 1, a.n_seqs, block_row);
            while (seq < a.n_seqs && a.q_starts[seq + 1] <= row) ++seq;   // a few rows behind block_row: rarely a step
        }
        const bool owned = live && seq < a.n_seqs;
        const int b = owned ? seq : 0;
        int64_t r0, r1;
        seq_rows(a.q_starts, b, a.rows, r0, r1);
        // counted back from the length as it is: a position from max_keys on has no place, and cutting the length first would
        // move its row onto a position that is there
        const int64_t at = a.seq_lens[b] - (r1 - row);
        const bool placed = at >= 0 && at < a.max_keys;
        const int c = placed ? (int)at : 0;
        pos = a.positions ? a.positions[row] : c;
        live = owned && row >= r0 && placed && pos >= 0;
        page = a.table.page(b, live ? c : 0);
        in_pool = ((((size_t)max(page, 0) * a.nk) << a.table.page_shift) + (c & ((1 << a.table.page_shift) - 1))) * D + i0;
    } else {
        pos = a.positions ? a.positions[row] : 0;
        live = live && pos >= 0;
    }

    // angles: cos / sin of the lane's four pairs (i, i + 1), or of its eight dimensions whose partners are half a rotation away
    const int half = a.rot.rotary_dim >> 1;
    const bool turns = i0 < a.rot.rotary_dim, pairs = a.rot.style == LCMHIP_ROTARY_PAIRS, first = i0 < half;
    const int lane = threadIdx.x & 63, partner = turns ? lane + (first ? half / 8 : -(half / 8)) : lane;
    float cs[8] = {}, sn[8] = {};
    if (turns) {
        const size_t at = (size_t)min(max(pos, 0), a.rot.n_positions - 1) * half + (pairs ? i0 >> 1 : (first ? i0 : i0 - half));
        if (pairs) {
            *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(a.rot.cos + at);
            *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(a.rot.sin + at);
        } else {
            load8<float>(a.rot.cos + at, cs);
            load8<float>(a.rot.sin + at, sn);
#pragma unroll
            for (int j = 0; j < 8; ++j) sn[j] = first ? -sn[j] : sn[j];
        }
    }

    auto transform = [&](const Raw8<T>& raw, const float (&w)[8], const void* bias, T* dst) {
        float x[8];
        load8<T>(reinterpret_cast<const T*>(&raw), x);
        if (a.norm.kind != LCMHIP_NORM_NONE) {
            if (a.norm.kind != LCMHIP_NORM_RMS) {
                float s = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += x[j];
                s = head_sum<LPH>(s) * (1.f / D);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] -= s;
            }
            float s2 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) s2 += x[j] * x[j];
            const float r = __builtin_amdgcn_rsqf(head_sum<LPH>(s2) * (1.f / D) + a.norm.eps);   // off by no more than 2^-23
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
            if (bias) {
                float t[8];
                load8<T>(reinterpret_cast<const T*>(bias) + i0, t);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] += t[j];
            }
        }
        if (a.rot.rotary_dim > 0) {
            if (pairs) {
                if (turns) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) rope_rotate(x[2 * j], x[2 * j + 1], cs[j], sn[j]);
                }
            } else {
                float y[8];
                if (LPH == 16 && half == 64) {             // eight lanes away: half a turn of the 16
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = dpp<0x128>(x[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = __shfl(x[j], partner, 64);
                }
                if (turns) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = x[j] * cs[j] + y[j] * sn[j];
                }
            }
            if (pos >= a.rot.n_positions) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_nanf("");
            }
        }
        store8<T>(dst, x);
    };
    // heads [h, end) of one kind: from `src` (of head 0 of the kind, which is head `base` of the row) to `dst`; null, for a row that
    // is skipped or whose page is not there: nothing is read
    auto heads = [&](int end, int base, const void* src, int64_t src_row, int64_t src_head, T* dst, int64_t dst_head, bool value,
                     const void* weight, const void* bias) {
        end = min(end, h1);
        if (!dst) {                                        // the same for all lanes of a head
            h += (max(end - h, 0) + hs - 1) >> head_shift << head_shift;
            return;
        }
        const T* from = reinterpret_cast<const T*>(src) + row * src_row + i0;
        float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (weight) load8<T>(reinterpret_cast<const T*>(weight) + i0, w);
        for (; h < end; h += CHUNK * hs) {
            Raw8<T> raw[CHUNK];
#pragma unroll
            for (int it = 0; it < CHUNK; ++it) {
                raw[it] = Raw8<T>{};
                if (h + it * hs < end) raw[it].load(from + (h + it * hs - base) * src_head);
            }
#pragma unroll
            for (int it = 0; it < CHUNK; ++it) {
                if (h + it * hs >= end) {                  // the same for all lanes of a head
                    h += it * hs;                          // the next kind begins here
                    return;
                }
                T* to = dst + (h + it * hs - base) * dst_head;
                if (!value) transform(raw[it], w, bias, to);
                else *reinterpret_cast<Raw8<T>*>(to) = raw[it];
            }
        }
    };
    T* k_dst;
    int64_t k_dst_head;
    if (APPEND) {
        k_dst = live && page >= 0 ? reinterpret_cast<T*>(a.k_pages) + in_pool : nullptr;
        k_dst_head = (int64_t)D << a.table.page_shift;
    } else {
        k_dst = live ? reinterpret_cast<T*>(a.k_out) + row * a.ko_row + i0 : nullptr;
        k_dst_head = a.ko_head;
    }
    heads(a.nq, 0, a.q, a.q_row, a.q_head, live ? reinterpret_cast<T*>(a.q_out) + row * a.qo_row + i0 : nullptr, a.qo_head, false,
          a.norm.q_weight, a.norm.q_bias);
    heads(a.nq + a.nk, a.nq, a.k, a.k_row, a.k_head, k_dst, k_dst_head, false, a.norm.k_weight, a.norm.k_bias);
    if (APPEND)
        heads(nh, a.nq + a.nk, a.v, a.v_row, a.v_head, live && page >= 0 ? reinterpret_cast<T*>(a.v_pages) + in_pool : nullptr, k_dst_head,
              true, nullptr, nullptr);
}

template <typename T, int D, bool APPEND>
static int launch_head_rows_t(const HeadArgs& a, hipStream_t st) {
    constexpr int SLOTS = 256 / (D / 8), WAVE_SLOTS = SLOTS / 4;
    const int nh = a.nq + a.nk + a.nv;
    if (a.rows == 0 || nh == 0) return LCMHIP_OK;
    // neighbouring heads in a wave: as many as leave fewest lane groups without one
    int shift = 0;
    auto rounded = [&](int s) { return ((nh + (1 << s) - 1) >> s) << s; };
    for (int s = 1; (1 << s) <= WAVE_SLOTS; ++s)
        if (rounded(s) <= rounded(shift)) shift = s;
    // a row's heads in one workgroup once the rows alone give the 256 CUs four workgroups each, else shared out over more
    const int64_t blocks = (a.rows + (SLOTS >> shift) - 1) / (SLOTS >> shift);
    const int turns = rounded(shift) >> shift;             // heads of a lane group, if one workgroup has them all
    int64_t shares = std::min<int64_t>(turns, std::max<int64_t>(1, 1024 / blocks));
    const int each = (int)((turns + shares - 1) / shares);
    shares = (turns + each - 1) / each;
    LCM_REQUIRE(blocks <= kMaxBlocks && shares <= 65535, "head rows: too many rows or heads, more workgroups than a launch holds");
    const dim3 grid((unsigned)blocks, (unsigned)shares);
    if (each > 1) hipLaunchKernelGGL((k_head_rows<T, D, APPEND, 4>), grid, dim3(256), 0, st, a, shift, each << shift);
    else hipLaunchKernelGGL((k_head_rows<T, D, APPEND, 1>), grid, dim3(256), 0, st, a, shift, each << shift);
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
    LCM_REQUIRE(!q || !rows_overlap(rows, n_heads, q_out_row, q_out_head, head_dim), "head_norm_rope: rows of q_out lie on each other");
    LCM_REQUIRE(!k || !rows_overlap(rows, n_kv_heads, k_out_row, k_out_head, head_dim), "head_norm_rope: rows of k_out lie on each other");
    HeadArgs a{};
    LCM_TRY(take_transform(a, norm, rotary, head_dim, q != nullptr, k != nullptr));
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.k = k; a.k_row = k_row; a.k_head = k_head;
    a.q_out = q_out; a.qo_row = q_out_row; a.qo_head = q_out_head;
    a.k_out = k_out; a.ko_row = k_out_row; a.ko_head = k_out_head;
    a.rows = rows; a.nq = q ? n_heads : 0; a.nk = k ? n_kv_heads : 0;
    a.positions = positions;
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
    if (batch->n_seqs == 0) return LCMHIP_OK;              // rows of no sequence
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
