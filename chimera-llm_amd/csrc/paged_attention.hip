// Attention of a ragged batch over the pages of its sequences, with or without prefixes that groups of sequences share.
//
//     o = sum_i exp(scale (x_i - m)) v_i / sum_i exp(scale (x_i - m)),   x_i = q . k_i,   m = max_i x_i
//
// in one pass over the keys with a running m, l = sum exp and o; two parts (m, l, o) of a row join as
//     m = max(m1, m2),   l = l1 w1 + l2 w2,   o = o1 w1 + o2 w2,   w = exp(scale (m_i - m)).
// The long axis is the keys': a sequence's keys are cut into parts that different workgroups walk, and k_paged_join joins
// them.  A prefix that sequences share is one more list of parts, whose rows are all rows of the group.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "paged.h"

namespace lcmhip {

using bf16x8_t = __attribute__((ext_vector_type(8))) __bf16;
using u32x4_t = __attribute__((ext_vector_type(4))) uint32_t;
using u32x2_t = __attribute__((ext_vector_type(2))) uint32_t;
using f32x4_t = __attribute__((ext_vector_type(4))) float;

// Lists of keys that rows attend to: a sequence's own positions, or the prefix of a group of sequences.
struct KeyLists {
    PageTable table;
    const int32_t* lens;
    const int32_t* group_starts;     // null: list i belongs to sequence i
    int n, max_keys;
    int causal;                      // row r of the list sees keys [0, len - rows + r + 1), of those that are there
    int splits, part0;               // parts of a list, and the number of the first
    int many, tiles;                 // many_rows(), and how many tiles of rows all lists have together
    int alone;                       // few_rows(): every wave has a part of its own (short parts), or four waves share one
};

struct PagedArgs {
    const void* q; int64_t q_row, q_head;
    void* out;
    const void *kp, *vp;
    const int32_t* q_starts;
    int n_seqs, rows, hq, hk;
    int G;                     // query heads of a key head
    uint32_t g_magic, g_shift; // x / G = (umulhi(g_magic, x) + x) >> g_shift for 0 <= x < 2^31
    float scale_log2;          // scale * log2(e).  It multiplies differences of dot products only: a product that fits fp32
                               // may leave it when multiplied by log2(e), and far from zero its rounding is no small number
    float* part_o;             // [part][row][head][D], not divided by l; null: a single part, finished in place
    float2* part_ml;           // [part][row][head] (m, l)
};

__device__ __forceinline__ int div_g(const PagedArgs& a, int x) { return (int)((__umulhi(a.g_magic, (uint32_t)x) + (uint32_t)x) >> a.g_shift); }

// Rows of list i, its length and how many of its keys are there.  Rows are counted back from the length: a list that is longer
// than max_keys ends in rows whose own positions are not there and which see all keys.
__device__ __forceinline__ void list_extent(const PagedArgs& a, const KeyLists& ls, int i, int& r0, int& r1, int& len, int& keys) {
    int s0 = i, s1 = i + 1;
    if (ls.group_starts) {
        s0 = min(max(read_index(ls.group_starts + i), 0), a.n_seqs);
        s1 = min(max(read_index(ls.group_starts + i + 1), s0), a.n_seqs);
    }
    r0 = a.q_starts ? read_index(a.q_starts + s0) : s0;
    r1 = a.q_starts ? read_index(a.q_starts + s1) : s1;
    r0 = min(max(r0, 0), a.rows);
    r1 = min(max(r1, r0), a.rows);
    len = max(0, read_index(ls.lens + i));
    keys = min(len, ls.max_keys);
}

constexpr int kMinPartFew = 256;   // keys a workgroup of k_paged_few is worth
// Part `split` of `keys` keys: at most `splits` equal parts, multiples of STEP keys, of no fewer than `least`.
template <int STEP>
__device__ __forceinline__ void part_range(int keys, int splits, int least, int split, int& k0, int& k1) {
    const int n = max(1, min(splits, (keys + least - 1) / least));
    const int len = ((keys + n - 1) / n + STEP - 1) / STEP * STEP;
    k0 = min(keys, split * len);
    k1 = min(keys, k0 + len);
}

// ---- a tile of 16 rows against groups of keys, by one wave ------------------------------------------------------------------
// Both products run on 16 x 16 matrix instructions with the keys (dims) as rows and the query rows as columns, so that a lane
// keeps one query row (lane % 16) throughout and softmax statistics need no exchange but over the four quads (lane / 16):
//     S^T[key][row] = K Q^T        lane holds keys 4 quad .. 4 quad + 3 of every 16
//     O^T[dim][row] += V^T P^T      the lane's own probabilities are its P^T operand
// The order of the inner index is free as long as both operands agree: key slots are numbered so that the operand P^T is
// what the lane holds, and dim rows so that the operand V^T is what 16-byte loads of value rows bring (below).
// No operand passes through LDS, and consecutive lanes read consecutive bytes.
__device__ __forceinline__ void store4(float* p, f32x4_t x) { *reinterpret_cast<f32x4_t*>(p) = x; }
__device__ __forceinline__ void store4(bf16_t* p, f32x4_t x) {
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{(uint32_t)f32_to_bf16(x[0]) | ((uint32_t)f32_to_bf16(x[1]) << 16),
                                             (uint32_t)f32_to_bf16(x[2]) | ((uint32_t)f32_to_bf16(x[3]) << 16)};
}

// Mask of the bf16 halves of a word that are NaN or infinite.
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
    return ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

template <typename T, int D>
struct Tile16;

template <int D>
struct Tile16<bf16_t, D> {
    static constexpr int kKeys = 32;                       // two 16-key halves, each in one page
    static constexpr int kHalves = 2;
    static constexpr int kO = D / 16;                      // accumulators; o[c][r] is dim kO * (4 quad + r) + c
    using vpiece_t = typename std::conditional<D == 128, u32x4_t, u32x2_t>::type;   // kO consecutive dims of a value row
    bf16x8_t q[D / 32], k[2][D / 32];
    vpiece_t v[2][4];                                      // value row 4 quad + e of half h, dims kO * (lane % 16) ..

    __device__ __forceinline__ void load_q(const bf16_t* row, bool live, int lane) {
#pragma unroll
        for (int st = 0; st < D / 32; ++st) {
            u32x4_t x = {0, 0, 0, 0};
            if (live) x = *reinterpret_cast<const u32x4_t*>(row + 32 * st + 8 * (lane >> 4));
            q[st] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    __device__ __forceinline__ void load_k(int h, const bf16_t* base, int lane) {
#pragma unroll
        for (int st = 0; st < D / 32; ++st)
            k[h][st] = *reinterpret_cast<const bf16x8_t*>(base + (lane & 15) * D + 32 * st + 8 * (lane >> 4));
    }
    __device__ __forceinline__ void load_v(int h, const bf16_t* base, int lane) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[h][e] = __builtin_nontemporal_load(reinterpret_cast<const vpiece_t*>(base + (4 * (lane >> 4) + e) * D + kO * (lane & 15)));
    }
    __device__ __forceinline__ void scores(float (&s)[8]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < D / 32; ++st) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[h][st], q[st], acc, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * h + e] = acc[e];
        }
    }
    __device__ __forceinline__ void clear_v(int h, int e) { v[h][e] = vpiece_t{}; }
    __device__ __forceinline__ bool v_not_finite(int h, int e) const {
        uint32_t bad = 0;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) bad |= not_finite(v[h][e][w]);
        return bad != 0;
    }
    // V^T operand c: dim kO * (lane % 16) + c of the lane's 8 value rows, picked out of the pieces that hold kO dims of one row
    __device__ __forceinline__ bf16x8_t v_operand(int c) const {
        const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
        u32x4_t x;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int p = 0; p < 2; ++p) x[2 * h + p] = __builtin_amdgcn_perm(v[h][2 * p + 1][c / 2], v[h][2 * p][c / 2], sel);
        return __builtin_bit_cast(bf16x8_t, x);
    }
    // A weight enters the second product as two bf16 numbers, its upper bits and the rest: the matrix unit has time for both while the
    // wave waits for memory.  The upper bits are cut, not rounded, and the rest gets 2^-24 of the weight more: both are positive
    // where the weight is, so that an infinite value stays one (a rest of 0, or below it, would make it NaN).  Cutting leaves a rest
    // below 2^-7 of the weight, whose own rounding is 2^-8 of that: 2^-15 of the weight is lost at most.
    __device__ __forceinline__ void weigh(const float (&p)[8], f32x4_t (&o)[kO]) const {
        u32x4_t cut;
        bf16x8_t rest;
#pragma unroll
        for (int e = 0; e < 8; ++e) rest[e] = (__bf16)fmaf(p[e], 0x1p-24f, p[e] - __uint_as_float(__float_as_uint(p[e]) & 0xffff0000u));
#pragma unroll
        for (int w = 0; w < 4; ++w) cut[w] = __builtin_amdgcn_perm(__float_as_uint(p[2 * w + 1]), __float_as_uint(p[2 * w]), 0x07060302u);
#pragma unroll
        for (int c = 0; c < kO; ++c) {
            const bf16x8_t x = v_operand(c);
            o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, rest, o[c], 0, 0, 0);
            o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8_t, cut), o[c], 0, 0, 0);
        }
    }
    // The values of key i that are not finite alone, into the rows (lanes) that see it.
    __device__ __forceinline__ void weigh_not_finite(const float (&p)[8], f32x4_t (&o)[kO], int i, bool visible, int lane) const {
        bf16x8_t pf;
#pragma unroll
        for (int e = 0; e < 8; ++e) pf[e] = (__bf16)p[e];
        const uint32_t mask = (lane >> 4) == ((i & 15) >> 2) ? ((i & 1) ? 0xffff0000u : 0x0000ffffu) : 0u;
        const int word = 2 * (i >> 4) + ((i & 3) >> 1);
#pragma unroll
        for (int c = 0; c < kO; ++c) {
            u32x4_t x = __builtin_bit_cast(u32x4_t, v_operand(c));
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] = w == word ? x[w] & not_finite(x[w]) & mask : 0u;
            const f32x4_t y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), pf, f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[c][r] += visible ? y[r] : 0.f;
        }
    }
    __device__ __forceinline__ void clear_not_finite() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < D / 32; ++w) v[h][e][w] &= ~not_finite(v[h][e][w]);
    }
    __device__ static __forceinline__ int dim(int c, int r, int lane) { return kO * (4 * (lane >> 4) + r) + c; }
};

template <int D>
struct Tile16<float, D> {
    static constexpr int kKeys = 16;
    static constexpr int kHalves = 1;
    static constexpr int kO = D / 16;                      // o[4 u + c][r] is dim 64 u + 4 (4 quad + r) + c
    f32x4_t q[D / 16], k[1][D / 16];                       // dims 16 i + 4 quad .. + 3
    f32x4_t v[1][4][D / 64];                               // value row 4 quad + e, dims 64 u + 4 (lane % 16) .. + 3

    __device__ __forceinline__ void load_q(const float* row, bool live, int lane) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            q[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (live) q[i] = *reinterpret_cast<const f32x4_t*>(row + 16 * i + 4 * (lane >> 4));
        }
    }
    __device__ __forceinline__ void load_k(int, const float* base, int lane) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) k[0][i] = *reinterpret_cast<const f32x4_t*>(base + (lane & 15) * D + 16 * i + 4 * (lane >> 4));
    }
    __device__ __forceinline__ void load_v(int, const float* base, int lane) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < D / 64; ++u)
                v[0][e][u] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(base + (4 * (lane >> 4) + e) * D + 64 * u + 4 * (lane & 15)));
    }
    __device__ __forceinline__ void scores(float (&s)[4]) const {
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0][i][e], q[i][e], acc, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = acc[e];
    }
    __device__ __forceinline__ void clear_v(int, int e) {
#pragma unroll
        for (int u = 0; u < D / 64; ++u) v[0][e][u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ bool v_not_finite(int, int e) const {
        bool bad = false;
#pragma unroll
        for (int u = 0; u < D / 64; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) bad |= not_finite(v[0][e][u][c]);
        return bad;
    }
    __device__ __forceinline__ void weigh(const float (&p)[4], f32x4_t (&o)[kO]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < D / 64; ++u)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[4 * u + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0][e][u][c], p[e], o[4 * u + c], 0, 0, 0);
    }
    __device__ __forceinline__ void weigh_not_finite(const float (&p)[4], f32x4_t (&o)[kO], int i, bool visible, int lane) const {
        const bool mine = (lane >> 4) == (i >> 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e != (i & 3)) continue;
#pragma unroll
            for (int u = 0; u < D / 64; ++u)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float x = v[0][e][u][c];
                    const f32x4_t y = __builtin_amdgcn_mfma_f32_16x16x4f32(mine && not_finite(x) ? x : 0.f, p[e], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[4 * u + c][r] += visible ? y[r] : 0.f;
                }
        }
    }
    __device__ __forceinline__ void clear_not_finite() {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int u = 0; u < D / 64; ++u)
#pragma unroll
                for (int c = 0; c < 4; ++c) v[0][e][u][c] = not_finite(v[0][e][u][c]) ? 0.f : v[0][e][u][c];
    }
    __device__ static __forceinline__ int dim(int c, int r, int lane) { return 64 * (c >> 2) + 4 * (4 * (lane >> 4) + r) + (c & 3); }
};

// Few rows for each list of keys: a tile of 16 (row, head of the group) pairs of one key head against one part of a list, four
// waves that take the part's groups of keys in turn and join their results in LDS (or, for short parts, a part for each wave).
// Bound by the bytes of the keys and values: with one row a list 15 of the 16 columns of a product are empty, and the matrix unit
// is still busy for less than a third of the time the bytes take.  Two rounds of loads are in flight for every wave (the values of
// this group, the keys of the next), 128 KB a CU.  One row for each of 64 documents of 1000-3800 keys, 16 heads, bf16: 208 us, 6.3
// TB/s; two sequences of 120k-131k keys, 8 key heads: 155 us and 5 for the join, 6.2 TB/s; one of 137 keys, fp32: 9.4 us a call, all
// of it the chain length -> page -> keys -> values -> join.  Each of its three rounds waits for its own keys: the next page id is
// looked up inside the loop and one group of keys is in flight.  Eight waves instead of four made that one slower (9.2 against 7.7 us
// launch to launch).
template <int D>
struct FewShared {
    float o[4][16][D + 4];
    float2 ml[4][16];
};
template <typename T, int D>
__device__ __forceinline__ void few_rows(const PagedArgs& a, const KeyLists& ls, int bid, FewShared<D>& red) {
    using Tile = Tile16<T, D>;
    constexpr int NP = 4 * Tile::kHalves;
    const int lane = threadIdx.x & 63, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int stride = ls.alone ? Tile::kKeys : 4 * Tile::kKeys;   // from one group of keys of this wave to the next
    if (ls.alone) {
        bid = 4 * bid + wave;
        if (bid >= a.hk * ls.splits * ls.n) return;        // no barrier below
    }
    const int hk = bid % a.hk;
    bid /= a.hk;
    const int split = bid % ls.splits;
    bid /= ls.splits;
    const int list = bid;
    const int G = a.G;
    int r0, r1, len, keys, k0, k1;
    list_extent(a, ls, list, r0, r1, len, keys);
    part_range<32>(keys, ls.splits, kMinPartFew, split, k0, k1);
    const int n_rows = (r1 - r0) * G;
    const T* kp = reinterpret_cast<const T*>(a.kp);
    const T* vp = reinterpret_cast<const T*>(a.vp);

    for (int t0 = 0; t0 < n_rows; t0 += 16) {              // more than one tile where a batch's max_q, or its average, said otherwise
        const int mine = t0 + (lane & 15);                 // (row, head) pair of this lane
        const bool live = mine < n_rows;
        const int token = live ? div_g(a, mine) : 0, row = r0 + token;
        const int head = hk * G + (live ? mine - token * G : 0);
        // keys that this row and the tile's first row see (later rows see no fewer)
        const int limit = ls.causal ? len - (r1 - row) + 1 : keys;
        const int first_limit = ls.causal ? len - (r1 - r0 - div_g(a, t0)) + 1 : keys;
        const int last_limit = ls.causal ? len - (r1 - r0 - div_g(a, min(t0 + 15, n_rows - 1))) + 1 : keys;
        const int end = min(k1, last_limit);

        Tile t;
        t.load_q(reinterpret_cast<const T*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.q_head, live, lane);
        f32x4_t o[Tile::kO];
#pragma unroll
        for (int c = 0; c < Tile::kO; ++c) o[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool seen = false;

        // place of the 16 keys from `key` on: element offset of the first, and how many of them there are
        auto place = [&](int key, size_t& off, int& there) {
            const int page = key < end ? ls.table.page(list, key) : -1;
            there = page >= 0 ? min(16, end - key) : 0;
            off = page >= 0 ? ((((size_t)page * a.hk + hk) << ls.table.page_shift) + (key & ((1 << ls.table.page_shift) - 1))) * D : 0;
        };
        size_t off[2], off_next[2];
        int there[2], there_next[2];
        int key = k0 + (ls.alone ? 0 : wave * Tile::kKeys);
#pragma unroll
        for (int h = 0; h < Tile::kHalves; ++h) {
            place(key + 16 * h, off[h], there[h]);
            if (key < end) t.load_k(h, kp + off[h], lane);
        }
        for (; key < end; key += stride) {
            // the values of this group and the keys of the next are in flight while the scores are worked out
#pragma unroll
            for (int h = 0; h < Tile::kHalves; ++h) t.load_v(h, vp + off[h], lane);
            const int next = key + stride;
#pragma unroll
            for (int h = 0; h < Tile::kHalves; ++h) place(next + 16 * h, off_next[h], there_next[h]);
            float s[NP];
            t.scores(s);
            if (next < end) {
#pragma unroll
                for (int h = 0; h < Tile::kHalves; ++h) t.load_k(h, kp + off_next[h], lane);
            }
            bool whole = key + Tile::kKeys <= first_limit;  // every row sees every key of the group
#pragma unroll
            for (int h = 0; h < Tile::kHalves; ++h) whole = whole && there[h] == 16;
            bool apart = false;                             // a hidden value is not finite: a product with 0 would show it
            if (whole) {
                seen = true;
            } else {
#pragma unroll
                for (int h = 0; h < Tile::kHalves; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * quad + e;
                        const bool here = i < there[h], vis = here && key + 16 * h + i < limit;
                        if (!vis) s[4 * h + e] = -INFINITY;
                        seen |= vis;
                        if (!here) t.clear_v(h, e);
                        else if (key + 16 * h + i >= first_limit) apart |= t.v_not_finite(h, e);
                    }
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < NP; ++i) top = fmaxf(top, s[i]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m)) {                           // else the running maxima stand and nothing is scaled
                const float mn = fmaxf(m, top);
                const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
                m = mn;
                l *= w;
#pragma unroll
                for (int c = 0; c < Tile::kO; ++c) o[c] *= w;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float p[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                p[i] = __builtin_amdgcn_exp2f((s[i] - ref) * a.scale_log2);
                l += p[i];
            }
            if (__any(apart)) {
                // what is not finite goes one key at a time into the rows that see it; the rest of the group as ever
#pragma unroll 1
                for (int i = 0; i < Tile::kKeys; ++i) t.weigh_not_finite(p, o, i, key + i < limit, lane);
                t.clear_not_finite();
            }
            t.weigh(p, o);
#pragma unroll
            for (int h = 0; h < Tile::kHalves; ++h) {
                off[h] = off_next[h];
                there[h] = there_next[h];
            }
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        int any = seen ? 1 : 0;
        any |= __shfl_xor(any, 16, 64);
        any |= __shfl_xor(any, 32, 64);
        // m: -inf only where no key was seen; keys that all score -inf leave l = 0, and 0 / 0 as the formula has it
        if (any && m == -INFINITY) m = -FLT_MAX;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < Tile::kO; ++c) red.o[wave][lane & 15][Tile::dim(c, r, lane)] = o[c][r];
        if (quad == 0) red.ml[wave][lane & 15] = make_float2(m, l);
        // the waves' results of a row together, or this wave's alone (LDS operations of one wave keep their order)
        if (ls.alone) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else __syncthreads();
        const int tile_rows = min(16, n_rows - t0), w0 = ls.alone ? wave : 0, w1 = ls.alone ? wave + 1 : 4;
        for (int i = ls.alone ? lane : threadIdx.x; i < tile_rows * (D / 4); i += ls.alone ? 64 : 256) {
            const int x = i / (D / 4), d4 = i % (D / 4) * 4;
            float M = -INFINITY;
            for (int w = w0; w < w1; ++w) M = fmaxf(M, red.ml[w][x].x);
            float L = 0.f;
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
            for (int w = w0; w < w1; ++w) {
                const float2 ml = red.ml[w][x];
                const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * a.scale_log2);
                L += ml.y * f;
                acc += *reinterpret_cast<const f32x4_t*>(&red.o[w][x][d4]) * f;
            }
            const int token = div_g(a, t0 + x);
            const size_t at = (size_t)(r0 + token) * a.hq + hk * G + (t0 + x - token * G);
            if (a.part_o) {
                const size_t part = (size_t)(ls.part0 + split) * ((size_t)a.rows * a.hq) + at;
                *reinterpret_cast<f32x4_t*>(a.part_o + part * D + d4) = acc;
                if (d4 == 0) a.part_ml[part] = make_float2(M, L);
            } else {
                store4(reinterpret_cast<T*>(a.out) + at * D + d4, M == -INFINITY ? f32x4_t{0.f, 0.f, 0.f, 0.f} : acc / L);
            }
        }
        if (ls.alone) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else __syncthreads();
    }
}

// ---- a tile of 32 rows against tiles of keys in LDS, by one wave -----------------------------------------------------------------
// The same two products on 32 x 32 matrix instructions; lane = row lane % 32, hi = lane / 32:
//     S^T  register r of a 32-key block holds key 8 (r / 4) + 4 hi + r % 4
//     O^T  register r of dim block t holds row 8 (r / 4) + 4 hi + r % 4 of the block
// Keys and values lie row-major in LDS, 16-byte pieces permuted inside a row (piece ^ swizzle(row)) so that the pieces one
// instruction reads from different rows lie in different banks; LDS-DMA fills a row's pieces in that order.
using f32x16_t = __attribute__((ext_vector_type(16))) float;
using s16x4_t = __attribute__((ext_vector_type(4))) short;
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;

template <typename T, int D>
struct Tile32;

template <int D>
struct Tile32<bf16_t, D> {
    static constexpr int kKeys = 64, kRow = 2 * D, kO = D / 32;
    bf16x8_t q[D / 16];
    int k_off, v_off[2];                                   // LDS byte offsets of this lane inside a tile, before the step's XOR

    // D = 128: a row is all 64 banks, so four consecutive rows go to four different quarters for the 8-byte transposed reads and
    // sixteen to sixteen pieces for the 16-byte reads.  D = 64: two rows are all banks.
    __device__ static __forceinline__ int swizzle(int row) {
        return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    }
    __device__ __forceinline__ void init(int lane) {
        const int c = lane & 31, hi = lane >> 5, i = lane & 15, dh = (lane >> 4) & 1;
        k_off = c * kRow + ((hi ^ swizzle(c)) << 4);       // piece 2 st + hi of row c: ^ (st << 5)
#pragma unroll
        for (int sec = 0; sec < 2; ++sec) {                // value rows 4 hi + i / 4 (+ 8), dims 16 dh + 4 (i % 4) ..: ^ (t << 6)
            const int row = 8 * sec + 4 * hi + (i >> 2);
            v_off[sec] = row * kRow + (((2 * dh + ((i & 3) >> 1)) ^ swizzle(row)) << 4) + 8 * (i & 1);
        }
    }
    // Keeps the offsets of all steps, one XOR each, from being worked out before the loop and held in registers.
    __device__ __forceinline__ void fresh_offsets() { asm volatile("" : "+v"(k_off), "+v"(v_off[0]), "+v"(v_off[1])); }
    __device__ __forceinline__ void load_q(const bf16_t* row, bool live, int lane) {
#pragma unroll
        for (int st = 0; st < D / 16; ++st) {
            u32x4_t x = {0, 0, 0, 0};
            if (live) x = *reinterpret_cast<const u32x4_t*>(row + 16 * st + 8 * (lane >> 5));
            q[st] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    __device__ __forceinline__ bf16x8_t k_operand(const char* ks, int kb, int st) const {   // dims 16 st + 8 hi .. of row lane % 32
        return *reinterpret_cast<const bf16x8_t*>(ks + kb * 32 * kRow + (k_off ^ (st << 5)));
    }
    __device__ __forceinline__ void scores(const char* ks, f32x16_t (&s)[2]) const {
        s[0] = s[1] = f32x16_t{};
#pragma unroll
        for (int st = 0; st < D / 16; ++st)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_operand(ks, kb, st), q[st], s[kb], 0, 0, 0);
    }
    __device__ __forceinline__ bf16x8_t v_operand(const char* vs, int kb, int u, int t) const {
        const char* base = vs + (kb * 32 + u * 16) * kRow;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(base + (v_off[0] ^ (t << 6))));
        const s16x4_t up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(base + (v_off[1] ^ (t << 6))));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // o += P V for a 32-key block.  Weights are rounded to bf16 (2^-8 of each at most, like the values they weigh; their sum is taken
    // before, in fp32): here the matrix unit is the bound, and the second product that Tile16 spends on what the rounding leaves takes
    // 588 us instead of 446 on eight prompts of 1500-2048 rows, 236 instead of 207 on 192 rows over prefixes of 20k-32k positions.
    __device__ __forceinline__ static bf16x8_t p_operand(const f32x16_t& p, int u) {
        bf16x8_t pf;
#pragma unroll
        for (int e = 0; e < 8; ++e) pf[e] = (__bf16)p[8 * u + e];
        return pf;
    }
    // One tile's weights and products, and the scores of the next: s[] holds the tile's scores and next[] takes the next one's.
    // A matrix instruction occupies its unit for 32 cycles (16 rows of 16 lanes a cycle would be 8 vector operations, 2 of them
    // exponentials): the exponentials of the first 32 keys stand between the products of the next scores, those of the other 32
    // between the products of the first 32 with their values, and every operand is read kAhead products ahead.  The order is pinned;
    // left alone the compiler puts all products before all exponentials.
    __device__ __forceinline__ void step(const char* ks_next, const char* vs, f32x16_t (&s)[2], f32x16_t (&next)[2], float c, float mc,
                                         float& l, f32x16_t (&o)[kO]) const {
        constexpr int kQ = D / 8, kV = 2 * kO;             // products of the scores; of 32 keys with their values
        constexpr int kPer = 16 / kQ, kPerV = 16 / kV;     // exponentials for each of them
        constexpr int kAhead = 4;                          // products whose operands are read ahead: an LDS read takes longer than three
        float sum[4] = {l, 0.f, 0.f, 0.f};
        auto weight = [&](int kb, int r) {
            s[kb][r] = __builtin_amdgcn_exp2f(fmaf(s[kb][r], c, -mc));
            sum[r & 3] += s[kb][r];
        };
        next[0] = next[1] = f32x16_t{};
        bf16x8_t ring[kAhead];
        auto operand = [&](int n) {                        // of product n: kQ for the scores, then kV for each half of the values
            if (n < kQ) return k_operand(ks_next, n & 1, n >> 1);
            return v_operand(vs, (n - kQ) / kV, (n - kQ) % kV / kO, (n - kQ) % kO);
        };
#pragma unroll
        for (int n = 0; n < kAhead; ++n) ring[n] = operand(n);
        bf16x8_t pf;
#pragma unroll
        for (int n = 0; n < kQ + 2 * kV; ++n) {
            if (n < kQ) {
                next[n & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[n % kAhead], q[n >> 1], next[n & 1], 0, 0, 0);
#pragma unroll
                for (int x = 0; x < kPer; ++x) weight(0, n * kPer + x);
            } else {
                const int kb = (n - kQ) / kV, i = (n - kQ) % kV;
                if (i % kO == 0) pf = p_operand(s[kb], i / kO);
                o[i % kO] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[n % kAhead], pf, o[i % kO], 0, 0, 0);
                if (kb == 0) {
#pragma unroll
                    for (int x = 0; x < kPerV; ++x) weight(1, i * kPerV + x);
                }
            }
            if (n + kAhead < kQ + 2 * kV) ring[n % kAhead] = operand(n + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    // Infinities and NaNs of a block's values for the rows that see them (bit r of `sees`: the key of register r): counted by a
    // product of ones, in which nothing can leave its row.
    __device__ __forceinline__ void add_not_finite(const char* vs, int kb, uint32_t sees, f32x16_t (&o)[kO]) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            bf16x8_t ones;
#pragma unroll
            for (int e = 0; e < 8; ++e) ones[e] = (__bf16)((sees >> (8 * u + e)) & 1 ? 1.f : 0.f);
#pragma unroll
            for (int t = 0; t < kO; ++t) {
                const u32x4_t x = __builtin_bit_cast(u32x4_t, v_operand(vs, kb, u, t));
#pragma unroll 1
                for (uint32_t sign = 0; sign < 2; ++sign) {    // the positive infinities and the NaNs, then the negative ones and the NaNs
                    u32x4_t y;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t lo = x[w] & 0xffffu, up = x[w] >> 16, inf = 0x7f80u | sign << 15;
                        y[w] = (lo == inf || (lo & 0x7fffu) > 0x7f80u ? 0x3f80u : 0u) | (up == inf || (up & 0x7fffu) > 0x7f80u ? 0x3f800000u : 0u);
                    }
                    const f32x16_t n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, y), ones, f32x16_t{}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[t][r] += n[r] > 0.f ? (sign ? -INFINITY : INFINITY) : 0.f;
                }
            }
        }
    }
    __device__ static __forceinline__ u32x4_t finite(u32x4_t x) {
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] &= ~not_finite(x[w]);
        return x;
    }
    // dims of registers 4 g .. 4 g + 3 of block t are consecutive
    __device__ static __forceinline__ void store(float* dst, const f32x16_t (&o)[kO], float f, int lane) {
#pragma unroll
        for (int t = 0; t < kO; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4_t*>(dst + 32 * t + 8 * g + 4 * (lane >> 5)) =
                    f32x4_t{o[t][4 * g] * f, o[t][4 * g + 1] * f, o[t][4 * g + 2] * f, o[t][4 * g + 3] * f};
    }
    __device__ static __forceinline__ void store(bf16_t* dst, const f32x16_t (&o)[kO], float f, int lane) {
#pragma unroll
        for (int t = 0; t < kO; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                u32x2_t x;
                x[0] = (uint32_t)f32_to_bf16(o[t][4 * g] * f) | ((uint32_t)f32_to_bf16(o[t][4 * g + 1] * f) << 16);
                x[1] = (uint32_t)f32_to_bf16(o[t][4 * g + 2] * f) | ((uint32_t)f32_to_bf16(o[t][4 * g + 3] * f) << 16);
                *reinterpret_cast<u32x2_t*>(dst + 32 * t + 8 * g + 4 * (lane >> 5)) = x;
            }
    }
};

template <int D>
struct Tile32<float, D> {
    static constexpr int kKeys = 32, kRow = 4 * D, kO = D / 32;
    f32x4_t q[D / 8];                                      // dims 8 i + 4 hi .. + 3
    int k_off, v_off;

    __device__ static __forceinline__ int swizzle(int row) { return row & 15; }
    __device__ __forceinline__ void init(int lane) {
        const int c = lane & 31, hi = lane >> 5;
        k_off = c * kRow + ((hi ^ swizzle(c)) << 4);       // piece 2 i + hi of row c: ^ (i << 5)
        v_off = 4 * hi * kRow + ((c * kO * 4) ^ (hi << 6)); // dims kO c .. of value row 4 hi, whose pieces are XORed with the key
    }
    __device__ __forceinline__ void fresh_offsets() { asm volatile("" : "+v"(k_off), "+v"(v_off)); }
    __device__ __forceinline__ void load_q(const float* row, bool live, int lane) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            q[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (live) q[i] = *reinterpret_cast<const f32x4_t*>(row + 8 * i + 4 * (lane >> 5));
        }
    }
    __device__ __forceinline__ void scores(const char* ks, f32x16_t (&s)[1]) const {
        s[0] = f32x16_t{};
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const f32x4_t k = *reinterpret_cast<const f32x4_t*>(ks + (k_off ^ (i << 5)));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[i][e], s[0], 0, 0, 0);
        }
    }
    using piece_t = typename std::conditional<D == 128, f32x4_t, __attribute__((ext_vector_type(2))) float>::type;
    __device__ __forceinline__ piece_t v_operand(const char* vs, int r) const {      // key 8 (r / 4) + 4 hi + r % 4
        return *reinterpret_cast<const piece_t*>(vs + (8 * (r >> 2) + (r & 3)) * kRow + (v_off ^ ((8 * (r >> 2 & 1) + (r & 3)) << 4)));
    }
    // As in bf16; 128 products of 64 cycles leave the order of the rest to the compiler.
    __device__ __forceinline__ void step(const char* ks_next, const char* vs, f32x16_t (&s)[1], f32x16_t (&next)[1], float c, float mc,
                                         float& l, f32x16_t (&o)[kO]) const {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[0][r] = __builtin_amdgcn_exp2f(fmaf(s[0][r], c, -mc));
            l += s[0][r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const piece_t v = v_operand(vs, r);
#pragma unroll
            for (int x = 0; x < kO; ++x) o[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[x], s[0][r], o[x], 0, 0, 0);
        }
        scores(ks_next, next);
    }
    __device__ __forceinline__ void add_not_finite(const char* vs, int, uint32_t sees, f32x16_t (&o)[kO]) const {
#pragma unroll
        for (int c = 0; c < kO; ++c) {
#pragma unroll 1
            for (int sign = 0; sign < 2; ++sign) {
                f32x16_t n = {};
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float v = v_operand(vs, r)[c];
                    const bool bad = not_finite(v) && !(sign ? v > 0.f : v < 0.f);
                    n = __builtin_amdgcn_mfma_f32_32x32x2f32(bad ? 1.f : 0.f, (sees >> r) & 1 ? 1.f : 0.f, n, 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) o[c][x] += n[x] > 0.f ? (sign ? -INFINITY : INFINITY) : 0.f;
            }
        }
    }
    __device__ static __forceinline__ u32x4_t finite(u32x4_t x) {
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] = not_finite(__uint_as_float(x[w])) ? 0u : x[w];
        return x;
    }
    // register r of block c is dim kO (8 (r / 4) + 4 hi + r % 4) + c
    __device__ static __forceinline__ void store(float* dst, const f32x16_t (&o)[kO], float f, int lane) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int c = 0; c < kO; ++c) dst[kO * (8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) + c] = o[c][r] * f;
    }
};

// 64 lanes bring 16 bytes each, from base + off[j] + 1024 j (base the same for the wave) to the 1024 bytes at LDS offset dst +
// 1024 j, for j < N.  Written in assembly because the compiler waits for every outstanding LDS-DMA before any LDS read, whatever
// it reads; nothing is returned in registers, and the waits for the data are the loop's own (s_waitcnt vmcnt before the
// barrier).  One block for all of them: M0, which says where in LDS they go, is set and used in it.
template <int N>
__device__ __forceinline__ void lds_dma(const char* base, const uint32_t (&off)[N], uint32_t dst) {
    static_assert(N == 1 || N == 2 || N == 4, "offsets are 12 bits");
    if constexpr (N == 1)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off[0]), "s"(base) : "memory", "m0");
    if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\tglobal_load_lds_dwordx4 %2, %3 offset:1024" ::"s"(dst),
                     "v"(off[0]), "v"(off[1]), "s"(base) : "memory", "m0");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %5\n\tglobal_load_lds_dwordx4 %2, %5 offset:1024\n\t"
                     "global_load_lds_dwordx4 %3, %5 offset:2*1024\n\tglobal_load_lds_dwordx4 %4, %5 offset:3*1024" ::"s"(dst),
                     "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(base) : "memory", "m0");
}

// Many rows for each list of keys (prompts; all rows of a group against its prefix): a tile of 128 (row, head of the group)
// pairs of one key head against one part of a list; wave w has pairs 32 w .., and the four share the keys and values that
// LDS-DMA brings one tile ahead.  Two workgroups a CU.
// Bound by the matrix instructions at the clock that the chip's power leaves them: a stream of them from registers on random data
// reaches 1500-1700 TFLOP/s in bf16, a large library product 1380, this kernel 1080 on 16384 rows that see 16384 keys, 1020 causal,
// 900 on eight causal prompts of 1500-2048 rows behind up to 2048 cached positions (438-451 us), where beginning and ending a
// workgroup and the tiles on the diagonal count.  Without the LDS-DMA that took 418 of then 470 us, without the exponentials as
// well 393, with nothing but the products 320.  Measured and left: eight waves that share 256 rows, with two to four buffers (465
// against 456 us, short prompts 139 against 112), the loop unrolled twice, operands read six or eight products ahead.
template <typename T, int D>
struct ManyShared {
    char kv[2][2][Tile32<T, D>::kKeys * Tile32<T, D>::kRow];   // [buffer][keys, values]
};
template <typename T, int D>
__device__ __forceinline__ void many_rows(const PagedArgs& a, const KeyLists& ls, int bid, ManyShared<T, D>& shared) {
    using Tile = Tile32<T, D>;
    constexpr int KT = Tile::kKeys, ROW = Tile::kRow, PIECES = ROW / 16, GROUPS = KT / 16;
    constexpr int RPI = 1024 / ROW, NI = KT / 4 / RPI;     // rows of one DMA instruction, instructions of a wave for a tile
    auto& smem = shared.kv;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.G;
    const int hk = bid % a.hk;                             // workgroups of one key head meet in the same L2 (8 XCDs, dealt in turn)
    bid /= a.hk;
    const int split = bid % ls.splits;
    // Tiles are numbered so that list i has those from floor(r0 G / 128) + i on, which leaves every list as many as it needs.
    // Late tiles first: under a causal mask they have the most keys.
    const int tile = ls.tiles - 1 - bid / ls.splits;
    // 64 lists at a time, a lane each; the first whose tiles do not end before this one
    int list = -1, r0 = 0, r1 = 0, len = 0, keys = 0, k0, k1;
    for (int first = 0; first < ls.n; first += 64) {
        int x0 = 0, x1 = 0, xl = 0, xk = 0;
        const bool is_list = first + lane < ls.n;
        if (is_list) list_extent(a, ls, first + lane, x0, x1, xl, xk);
        const int c = __popcll(__ballot(is_list && (int)((int64_t)x1 * G >> 7) + first + lane + 1 <= tile));
        if (c < min(64, ls.n - first)) {
            list = first + c;
            r0 = __builtin_amdgcn_readlane(x0, c);
            r1 = __builtin_amdgcn_readlane(x1, c);
            len = __builtin_amdgcn_readlane(xl, c);
            keys = min(len, ls.max_keys);
            break;
        }
    }
    if (list < 0) return;
    part_range<KT>(keys, ls.splits, 2 * KT, split, k0, k1);
    const int n_rows = (r1 - r0) * G;
    const int t0 = (tile - (int)((int64_t)r0 * G >> 7) - list) * 128;
    if (t0 < 0 || t0 >= n_rows) return;

    const int mine = t0 + 32 * wave + (lane & 31);
    const bool live = mine < n_rows;
    const int token = live ? div_g(a, mine) : 0, row = r0 + token;
    const int head = hk * G + (live ? mine - token * G : 0);
    const int at_end = len - (r1 - r0) + 1;                // keys that the list's first row sees, if they are there
    const int limit = ls.causal ? len - (r1 - row) + 1 : keys;
    const int tile_end = min(k1, ls.causal ? at_end + div_g(a, min(t0 + 127, n_rows - 1)) : keys);
    const int tile_first = ls.causal ? at_end + div_g(a, t0) : keys;
    const bool wave_live = t0 + 32 * wave < n_rows;
    const int wave_first = ls.causal ? at_end + div_g(a, min(t0 + 32 * wave, n_rows - 1)) : keys;
    const int wave_end = !wave_live ? 0 : min(k1, ls.causal ? at_end + div_g(a, min(t0 + 32 * wave + 31, n_rows - 1)) : keys);

    Tile t;
    t.init(lane);
    t.load_q(reinterpret_cast<const T*>(a.q) + (int64_t)row * a.q_row + (int64_t)head * a.q_head, live, lane);
    f32x16_t o[Tile::kO];
#pragma unroll
    for (int c = 0; c < Tile::kO; ++c) o[c] = f32x16_t{};
    float m = -INFINITY, l = 0.f;
    bool seen = false;

    // Lane i holds the id of page page0 + i of the list: one load for 64 pages, a lane read for each use.  (Scalar loads inside
    // the loop would make every wait for an LDS read a wait for all of them.)  bad: the lanes whose page is not there.
    int page0 = k0 >> ls.table.page_shift, page_ids = 0;
    uint64_t bad = 0;
    auto load_ids = [&]() {
        const int at = (page0 + lane) << ls.table.page_shift;
        page_ids = ls.table.page(list, at);
        bad = __ballot(page_ids < 0 && at < tile_end);
    };
    // Bytes from the pool's begin to the 16-key group of tile kt that holds the rows this wave brings (rows wave * KT / 4 ..); where
    // the page is not there, to the pool's first group.
    const int my_group = wave * (KT / 4) & ~15;
    const uint64_t page_bytes = ((uint64_t)a.hk << ls.table.page_shift) * ROW, head_bytes = ((uint64_t)hk << ls.table.page_shift) * ROW;
    auto source_of = [&](int kt) {
        if (((kt + KT - 1) >> ls.table.page_shift) - page0 >= 64) {
            page0 = kt >> ls.table.page_shift;
            load_ids();
        }
        const int key = kt + my_group, id = __builtin_amdgcn_readlane(page_ids, (key >> ls.table.page_shift) - page0);
        const uint32_t in_page = (key & ((1 << ls.table.page_shift) - 1)) * ROW;
        return id < 0 ? head_bytes : (uint64_t)id * page_bytes + head_bytes + in_page;
    };
    // the 16-key groups of tile kt whose page is not there (kt no earlier than the pages held)
    auto absent_of = [&](int kt) {
        uint32_t x = 0;
        if (bad) {
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                x |= kt + 16 * g < tile_end && __builtin_amdgcn_readlane(page_ids, ((kt + 16 * g) >> ls.table.page_shift) - page0) < 0 ? 1u << g : 0u;
        }
        return x;
    };
    uint32_t dma_off[NI];                                  // of row j RPI + lane / PIECES behind the wave's first, less 1024 j
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int r = wave * (KT / 4) + j * RPI + lane / PIECES;
        dma_off[j] = (r & 15) * ROW + (((lane % PIECES) ^ Tile::swizzle(r)) << 4) - 1024 * j;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)&smem[0][0][0] + wave * (KT / 4) * ROW;
    auto request = [&](const void* pool, uint64_t source, int buf, int which) {
        lds_dma<NI>(reinterpret_cast<const char*>(pool) + source, dma_off, lds0 + (2 * buf + which) * (KT * ROW));
    };

    // Step i works on the scores of tile i, which step i - 1 left in registers, the values of tile i and the keys of tile i + 1;
    // meanwhile the values of tile i + 1 and the keys of tile i + 2 arrive.  Two buffers each, one barrier a step.
    f32x16_t s[KT / 32];
    const float grown = 8.f / a.scale_log2;                // weights may reach 2^8 before the running maximum is moved
    uint32_t absent0 = 0, absent1 = 0;                     // of tiles i and i + 1
    uint64_t source1 = 0;                                  // of tile i + 1
    if (k0 < tile_end) {
        load_ids();
        const uint64_t source0 = source_of(k0);
        request(a.kp, source0, 0, 0);
        request(a.vp, source0, 0, 1);
        absent0 = absent_of(k0);
        source1 = source_of(k0 + KT);
        absent1 = absent_of(k0 + KT);
        if (k0 + KT < tile_end) request(a.kp, source1, 1, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        t.scores(smem[0][0], s);
    }
    int buf = 0;
    for (int kt = k0; kt < tile_end; kt += KT) {
        // keys i + 1 and values i have landed, and every wave is done with the buffers of keys i and values i - 1
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        char* vs = smem[buf][1];
        const uint32_t absent = absent0;
        // Some keys are not there, or some rows of the workgroup do not see all of them: look for values that are not finite,
        // whose product with a weight of 0 would not be 0.
        bool apart = false;
        if (absent != 0 || kt + KT > min(tile_first, tile_end)) {
#pragma unroll 1
            for (int i = threadIdx.x * 16; i < KT * ROW; i += 4096) {
                const u32x4_t x = *reinterpret_cast<const u32x4_t*>(vs + i), y = Tile::finite(x);
                apart |= x[0] != y[0] || x[1] != y[1] || x[2] != y[2] || x[3] != y[3];
            }
            apart = __syncthreads_or(apart);
        }
        if (kt + KT < tile_end) request(a.vp, source1, buf ^ 1, 1);
        source1 = source_of(kt + 2 * KT);
        absent0 = absent1;
        absent1 = absent_of(kt + 2 * KT);
        if (kt + 2 * KT < tile_end) request(a.kp, source1, buf, 0);

        const bool active = kt < wave_end;
        uint32_t sees[KT / 32];
        if (absent != 0 || kt + KT > min(wave_first, tile_end)) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
                sees[kb] = 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = 32 * kb + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                    const bool vis = kt + i < limit && kt + i < tile_end && !(absent >> (i >> 4) & 1);
                    if (!vis) s[kb][r] = -INFINITY;
                    sees[kb] |= vis ? 1u << r : 0u;
                }
                seen |= sees[kb] != 0;
            }
        } else {
            seen |= active;
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) sees[kb] = 0xffffu;
        }
        if (active) {
            float top = s[0][0];
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
            const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
            if (__any(top > m + grown)) {                  // else no weight leaves [0, 2^8] and nothing is scaled
                const float mn = fmaxf(m, top);
                const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
                m = mn;
                l *= w;
#pragma unroll
                for (int c = 0; c < Tile::kO; ++c) o[c] *= w;
            }
        }
        if (__builtin_expect(apart, 0)) {
            if (active) {
#pragma unroll
                for (int kb = 0; kb < KT / 32; ++kb) t.add_not_finite(vs, kb, sees[kb], o);
            }
            __syncthreads();
#pragma unroll 1
            for (int i = threadIdx.x * 16; i < KT * ROW; i += 4096)
                *reinterpret_cast<u32x4_t*>(vs + i) = Tile::finite(*reinterpret_cast<const u32x4_t*>(vs + i));
            __syncthreads();
        }
        if (active) {
            // exp2(c x - c m) with one operation a score; far from zero, where the rounding of c m is no small number, m is
            // taken off first
            float mc = m == -INFINITY ? 0.f : m * a.scale_log2;
            if (__any(!(fabsf(mc) < 16384.f))) {
#pragma unroll
                for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] -= m == -INFINITY ? 0.f : m;
                mc = 0.f;
            }
            t.fresh_offsets();
            f32x16_t next[KT / 32];
            t.step(smem[buf ^ 1][0], vs, s, next, a.scale_log2, mc, l, o);   // behind the last tile: scores that nobody reads
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) s[kb] = next[kb];
        }
        buf ^= 1;
    }

    l += __shfl_xor(l, 32, 64);
    int any = seen ? 1 : 0;
    any |= __shfl_xor(any, 32, 64);
    if (any && m == -INFINITY) m = -FLT_MAX;               // as in k_paged_few
    if (!live) return;
    const size_t at = (size_t)row * a.hq + head;
    if (a.part_o) {
        const size_t part = (size_t)(ls.part0 + split) * ((size_t)a.rows * a.hq) + at;
        Tile::store(a.part_o + part * D, o, 1.f, lane);
        if (lane < 32) a.part_ml[part] = make_float2(m, l);
    } else {
        Tile::store(reinterpret_cast<T*>(a.out) + at * D, o, any ? 1.f / l : 0.f, lane);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_paged_few(PagedArgs a, KeyLists ls) {
    __shared__ FewShared<D> shared;
    few_rows<T, D>(a, ls, blockIdx.x, shared);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_paged_many(PagedArgs a, KeyLists ls) {
    __shared__ __attribute__((aligned(1024))) ManyShared<T, D> shared;
    many_rows<T, D>(a, ls, blockIdx.x, shared);
}

// Prefixes and own positions in one launch: small calls save one, and in large ones the prefixes, bound by matrix instructions, share
// the chip with own positions, bound by memory, as they run out.  n0 workgroups of `prefix`, then (from a multiple of 8 on: the
// XCDs are dealt in turn) n1 of `own`.  Spreading the two evenly instead took 225 us against 207 (192 continuations of four
// prefixes of 20k-32k positions).
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_paged_pair(PagedArgs a, KeyLists prefix, KeyLists own, int n0, int n1) {
    __shared__ __attribute__((aligned(1024))) union { FewShared<D> few; ManyShared<T, D> many; } shared;
    const int first_own = (n0 + 7) & ~7;
    const bool is_prefix = (int)blockIdx.x < first_own;
    const int bid = is_prefix ? blockIdx.x : blockIdx.x - first_own;
    if (bid >= (is_prefix ? n0 : n1)) return;
    const KeyLists& ls = is_prefix ? prefix : own;
    if (ls.many) many_rows<T, D>(a, ls, bid, shared.many);
    else few_rows<T, D>(a, ls, bid, shared.few);
}

struct JoinArgs {
    int parts, prefix_parts;         // the prefix's parts come first
    const int32_t* group_starts;     // null: no prefix
    int n_groups;
};

// Joins the parts of every (row, head).  D / 4 lanes hold a row's values; PG such groups take the parts in turn and meet in LDS
// (many parts of few rows), or one group takes them all (PG = 1).  Latency is all there is to it: 4-5 us a launch where loads
// depended on the weight of the part before took 39 (64 parts of 64 rows).
template <typename T, int D, int PG>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, JoinArgs j) {
    constexpr int L4 = D / 4, ROWS = 256 / L4 / PG, U = 8;
    __shared__ f32x4_t red_o[PG > 1 ? 256 : 1];
    __shared__ float2 red_ml[PG > 1 ? 256 / L4 : 1];
    const int sub = threadIdx.x % L4, group = threadIdx.x / L4, pg = group % PG;
    const int64_t at = (int64_t)blockIdx.x * ROWS + group / PG;
    const int64_t row = at / a.hq;
    // rows of no sequence are left alone; those of no group have no prefix
    const int first = a.q_starts ? read_index(a.q_starts) : 0, last = a.q_starts ? read_index(a.q_starts + a.n_seqs) : a.n_seqs;
    const bool live = row < a.rows && row >= first && row < last;
    int part0 = j.prefix_parts;
    if (j.group_starts) {
        const int s0 = min(max(read_index(j.group_starts), 0), a.n_seqs), s1 = min(max(read_index(j.group_starts + j.n_groups), 0), a.n_seqs);
        if (row >= (a.q_starts ? read_index(a.q_starts + s0) : s0) && row < (a.q_starts ? read_index(a.q_starts + s1) : s1)) part0 = 0;
    }
    const int64_t stride = (int64_t)a.rows * a.hq;
    float m = -INFINITY, l = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    // U parts at a time: all their loads are in flight before the first is used
    for (int p0 = live ? part0 + pg : j.parts; p0 < j.parts; p0 += U * PG) {
        float2 ml[U];
        f32x4_t o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t x = min(p0 + u * PG, j.parts - 1) * stride + at;
            ml[u] = a.part_ml[x];
            o[u] = *reinterpret_cast<const f32x4_t*>(a.part_o + x * D + 4 * sub);
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p0 + u * PG >= j.parts) ml[u].x = -INFINITY;
            mn = fmaxf(mn, ml[u].x);
        }
        const float w0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
        l *= w0;
        acc *= w0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (ml[u].x == -INFINITY) continue;            // an empty part wrote no values
            const float w = __builtin_amdgcn_exp2f((ml[u].x - mn) * a.scale_log2);
            l += ml[u].y * w;
            acc += o[u] * w;
        }
        m = mn;
    }
    if (PG > 1) {
        red_o[threadIdx.x] = acc;
        if (sub == 0) red_ml[group] = make_float2(m, l);
        __syncthreads();
        if (pg != 0) return;
        float M = -INFINITY;
#pragma unroll
        for (int g = 0; g < PG; ++g) M = fmaxf(M, red_ml[group + g].x);
        l = 0.f;
        acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < PG; ++g) {
            const float2 ml = red_ml[group + g];
            const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * a.scale_log2);
            l += ml.y * w;
            acc += red_o[threadIdx.x + g * L4] * w;
        }
        m = M;
    }
    if (live) {
        store4(reinterpret_cast<T*>(a.out) + at * D + 4 * sub, m == -INFINITY ? f32x4_t{0.f, 0.f, 0.f, 0.f} : acc / l);
    }
}

static int check_prefix(const lcmhip_kv_pages* pages, const lcmhip_shared_prefix* prefix) {
    LCM_REQUIRE(prefix && prefix->page_table && prefix->lens && prefix->group_starts, "shared prefix: null argument");
    LCM_REQUIRE(prefix->n_groups >= 1 && prefix->n_groups <= (1 << 24), "shared prefix: n_groups out of range");
    LCM_REQUIRE(prefix->max_pages >= 1, "shared prefix: max_pages must be positive");
    LCM_REQUIRE(prefix->max_keys >= 1 && prefix->max_keys <= kMaxKeys && prefix->max_keys <= (int64_t)prefix->max_pages * pages->page_size,
                "shared prefix: max_keys must be in [1, max_pages * page_size], at most 2^30");
    return LCMHIP_OK;
}

static int check_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, int64_t rows, int n_heads) {
    LCM_TRY(check_pages(pages));
    LCM_TRY(check_batch(pages, batch, rows));
    LCM_REQUIRE(n_heads >= 1 && n_heads <= 65535 && n_heads % pages->n_kv_heads == 0,
                "paged attention: n_heads must be a multiple of n_kv_heads");
    LCM_REQUIRE(rows * n_heads <= INT32_MAX - 1024, "paged attention: too many rows");
    return LCMHIP_OK;
}

// How a call is cut.  A list of keys goes to few_rows() where its rows fill no more than one tile of 16, else to many_rows(): 64
// lists of 2048 keys with 16 rows a key head take 104 / 98 us (few / many, bf16) and 211 / 301 us (fp32), with 32 rows 189 / 99 us
// and 387 / 292 us.
// few: parts are added until the grid has kWantedFew workgroups, eight for each place on the chip, so that lists of unequal
//      length even out (64 lists of 1000-3800 keys: 238 us with 2048 workgroups, 231 with 4096 or 8192).
//      With a right max_q these are at most 16 kWantedFew partial (row, head) results; a max_q that understates the rows would have up
//      to 64 for every row of the batch (16 GiB for 16384 rows of 32 heads of 128), so parts stop at kMaxPartials (0.5 GiB), which
//      leaves batches with up to 16 times as many padding rows as they are.
// many: a part takes a workgroup a step for each tile of keys and 3 us to begin and end, a round of kPlaces workgroups at a time,
//      and its rows' partial results are written and read once (about 3 TB/s); the number of parts that makes the sum least.
//      Twelve parts of a prefix of 3701 positions for 64 rows: 31.7 us, 4 parts 38.3, 32 parts 34.7.
constexpr int kWantedFew = 4096, kPlaces = 512, kMaxParts = 64, kMaxPartials = 1 << 20;
struct ListPlan {
    bool many = false, alone = false;
    int tiles = 0;             // many: tiles of rows in all
    int splits = 0;
};
struct Plan {
    ListPlan own, prefix;
    bool joined = false;
    size_t ml_bytes = 0, bytes = 0;
};

static ListPlan plan_lists(int64_t lists, int64_t list_rows, int64_t all_rows, int hk, int max_keys, int head_dim, int dtype) {
    ListPlan p;
    p.many = list_rows > 16;
    if (!p.many) {
        const int64_t most = std::min<int64_t>(kMaxParts, (max_keys + kMinPartFew - 1) / kMinPartFew);
        p.splits = (int)std::max<int64_t>(1, std::min({most, kWantedFew / (lists * hk), kMaxPartials / (all_rows * hk)}));
        // a wave for a part where four would have a group or two of keys each, once that still leaves every CU a workgroup
        p.alone = max_keys <= (int64_t)kMinPartFew * p.splits && lists * hk * p.splits >= 1024;
        return p;
    }
    p.tiles = (int)(all_rows / 128 + lists);
    // workgroups of one part, if the lists have about as many rows each
    const int64_t blocks = hk * std::max((all_rows + 127) / 128, lists * ((all_rows / lists + 127) / 128));
    const int step_keys = dtype == LCMHIP_BF16 ? 64 : 32;
    // Two workgroups a CU at the matrix unit's nominal rate.  512 workgroups do 2.15 GFLOP in a bf16 step, which the kernel does in
    // 2.0-2.4 us when the chip is full: joins and the fixed 3 us weigh about twice too much in large bf16 calls.
    const double step_us = (dtype == LCMHIP_BF16 ? 0.9 : 6.8) * head_dim / 128;
    const double join_us = (double)all_rows * hk * head_dim * 8 / 3e6;
    const int most = std::min(kMaxParts, (max_keys + 2 * step_keys - 1) / (2 * step_keys));
    double best = 0;
    for (int s = 1; s <= most; ++s) {
        const int64_t rounds = (blocks * s + kPlaces - 1) / kPlaces, steps = (max_keys + (int64_t)s * step_keys - 1) / ((int64_t)s * step_keys);
        const double cost = (double)rounds * (steps * step_us + 3.0) + (s > 1 ? 4.0 + s * join_us : 0.0);
        if (s == 1 || cost < best) {
            best = cost;
            p.splits = s;
        }
    }
    return p;
}

static Plan make_plan(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const lcmhip_shared_prefix* prefix, int64_t rows,
                      int n_heads) {
    Plan p;
    const int64_t G = n_heads / pages->n_kv_heads;
    if (batch->n_seqs == 0 || rows == 0) return p;
    p.own = plan_lists(batch->n_seqs, std::min<int64_t>(batch->max_q, rows) * G, rows * G, pages->n_kv_heads, batch->max_keys, pages->head_dim, pages->dtype);
    if (prefix)
        p.prefix = plan_lists(prefix->n_groups, (rows + prefix->n_groups - 1) / prefix->n_groups * G, rows * G, pages->n_kv_heads, prefix->max_keys, pages->head_dim, pages->dtype);
    p.joined = p.own.splits + p.prefix.splits > 1;
    if (p.joined) {
        const size_t n = (size_t)(p.own.splits + p.prefix.splits) * rows * n_heads;
        p.ml_bytes = (n * sizeof(float2) + 255) & ~(size_t)255;
        p.bytes = p.ml_bytes + n * pages->head_dim * sizeof(float);
    }
    return p;
}

template <typename T, int D>
static int launch_paged(const PagedArgs& a, const KeyLists& own, const KeyLists& prefix, const Plan& p, hipStream_t st) {
    auto blocks_of = [&](const KeyLists& ls) {
        const int64_t parts = (int64_t)a.hk * ls.splits * (ls.many ? ls.tiles : ls.n);
        return ls.alone ? (parts + 3) / 4 : parts;
    };
    const int64_t n1 = blocks_of(own), n0 = prefix.n > 0 ? blocks_of(prefix) : 0, pair = (((n0 + 7) >> 3) + ((n1 + 7) >> 3)) << 3;
    // joining: one group of lanes for a row while the rows alone fill the chip, else eight
    const JoinArgs j{p.own.splits + p.prefix.splits, p.prefix.splits, prefix.group_starts, prefix.n};
    const int64_t heads = (int64_t)a.rows * a.hq, per = 256 / (D / 4);
    const bool wide = heads / per >= 256 || j.parts <= 8;
    const int64_t n_join = wide ? (heads + per - 1) / per : (heads + per / 8 - 1) / (per / 8);
    LCM_REQUIRE((prefix.n > 0 ? pair : n1) <= kMaxBlocks && (!p.joined || n_join <= kMaxBlocks),
                "paged attention: too many rows or sequences, more workgroups than a launch holds");
    if (prefix.n > 0) {
        hipLaunchKernelGGL((k_paged_pair<T, D>), dim3((unsigned)pair), dim3(256), 0, st, a, prefix, own, (int)n0, (int)n1);
    } else if (own.many) {
        hipLaunchKernelGGL((k_paged_many<T, D>), dim3((unsigned)n1), dim3(256), 0, st, a, own);
    } else {
        hipLaunchKernelGGL((k_paged_few<T, D>), dim3((unsigned)n1), dim3(256), 0, st, a, own);
    }
    LCM_HIP_CHECK(hipGetLastError());
    if (p.joined) {
        if (wide) hipLaunchKernelGGL((k_paged_join<T, D, 1>), dim3((unsigned)n_join), dim3(256), 0, st, a, j);
        else hipLaunchKernelGGL((k_paged_join<T, D, 8>), dim3((unsigned)n_join), dim3(256), 0, st, a, j);
        LCM_HIP_CHECK(hipGetLastError());
    }
    return LCMHIP_OK;
}

static int paged_attention(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, const lcmhip_shared_prefix* prefix,
                           const void* q, int64_t q_row, int64_t q_head, void* out, int64_t rows, int n_heads, float scale,
                           int causal, void* ws, size_t ws_bytes, hipStream_t st) {
    LCM_TRY(check_attention(pages, batch, rows, n_heads));
    if (prefix) LCM_TRY(check_prefix(pages, prefix));
    LCM_REQUIRE(q && out, "paged attention: null argument");
    LCM_REQUIRE(scale >= 1e-20f && scale <= 1e20f, "paged attention: scale must lie in [1e-20, 1e20]");
    LCM_TRY(check_rows(q, q_row, q_head, pages->dtype, "paged attention: q"));
    LCM_TRY(check_rows(out, 0, 0, pages->dtype, "paged attention: out"));
    if (rows == 0 || batch->n_seqs == 0) return LCMHIP_OK;
    const Plan p = make_plan(pages, batch, prefix, rows, n_heads);
    LCM_REQUIRE(ws_bytes >= p.bytes && (p.bytes == 0 || (ws && (uintptr_t)ws % 256 == 0)),
                "paged attention: workspace too small, missing or not 256-byte aligned");
    PagedArgs a{};
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.out = out; a.kp = pages->k; a.vp = pages->v;
    a.q_starts = batch->q_starts; a.n_seqs = batch->n_seqs;
    a.rows = (int)rows; a.hq = n_heads; a.hk = pages->n_kv_heads; a.G = n_heads / pages->n_kv_heads;
    while ((1 << a.g_shift) < a.G) ++a.g_shift;
    a.g_magic = (uint32_t)((((uint64_t)1 << 32) * ((1u << a.g_shift) - a.G)) / a.G + 1);
    a.scale_log2 = scale * 1.4426950408889634f;
    const KeyLists own{PageTable{batch->page_table, batch->max_pages, page_shift_of(pages), (uint32_t)pages->n_pages}, batch->seq_lens, nullptr,
                     batch->n_seqs, batch->max_keys, causal != 0, p.own.splits, p.prefix.splits, p.own.many, p.own.tiles, p.own.alone};
    KeyLists pre{};
    if (prefix)
        pre = KeyLists{PageTable{prefix->page_table, prefix->max_pages, page_shift_of(pages), (uint32_t)pages->n_pages}, prefix->lens,
                            prefix->group_starts, prefix->n_groups, prefix->max_keys, 0, p.prefix.splits, 0, p.prefix.many, p.prefix.tiles, p.prefix.alone};
    if (p.joined) {
        a.part_ml = reinterpret_cast<float2*>(ws);
        a.part_o = reinterpret_cast<float*>(static_cast<char*>(ws) + p.ml_bytes);
    }
    if (pages->dtype == LCMHIP_BF16) return pages->head_dim == 64 ? launch_paged<bf16_t, 64>(a, own, pre, p, st) : launch_paged<bf16_t, 128>(a, own, pre, p, st);
    return pages->head_dim == 64 ? launch_paged<float, 64>(a, own, pre, p, st) : launch_paged<float, 128>(a, own, pre, p, st);
}

}  // namespace lcmhip

using namespace lcmhip;

extern "C" {

int lcmhip_paged_attention_workspace(const lcmhip_kv_pages* pages, const lcmhip_paged_batch* batch, int64_t rows, int32_t n_heads,
                                     size_t* bytes) {
    LCM_REQUIRE(bytes, "paged_attention_workspace: null argument");
    LCM_TRY(check_attention(pages, batch, rows, n_heads));
    *bytes = make_plan(pages, batch, nullptr, rows, n_heads).bytes;
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
    *bytes = make_plan(pages, batch, prefix, rows, n_heads).bytes;
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
