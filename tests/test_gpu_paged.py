"""The paged cache operators (lcm.nn.paged_attention) against their 64-bit statements (tests/paged_reference.py)."""

import math
import random

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def pa():
    assert torch.cuda.is_available()
    from lcm.nn import paged_attention
    return paged_attention


def _randn(g, *shape, dtype=F32, gain=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * gain).to(dtype)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _within(got, want, bound, what=""):
    assert torch.isfinite(got).all(), what
    over = (got.double() - want).abs() - bound
    i = int(over.argmax())
    assert float(over.max()) <= 0, (what, i, float(got.flatten()[i]), float(want.flatten()[i]), float(bound.flatten()[i]))


def _tables(pa, rot, style, n=4096):
    rope = pa.RotaryTable.create(n, rot, style=style)
    return rope, rope.cos, rope.sin


def _norm(pa, g, kind, d, dtype, bias=True):
    if kind is None:
        return None, (None,) * 4
    if kind == "unit":
        return pa.HeadNorm("unit"), (None,) * 4
    qw, kw = (1 + _randn(g, d, gain=0.2)).to(dtype), (1 + _randn(g, d, gain=0.2)).to(dtype)
    qb, kb = (_randn(g, d, gain=0.2).to(dtype), _randn(g, d, gain=0.2).to(dtype)) if kind == "standard" and bias else (None, None)
    return pa.HeadNorm(kind, qw, kw, qb, kb), (qw, kw, qb, kb)


# ---- norm and rotation of heads -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,hq,hk,d,kind,rot,style", [
    (1, 1, 1, 128, "rms", 128, "pairs"), (1, 16, 16, 128, None, 128, "halves"), (3, 5, 1, 64, "standard", 64, "halves"),
    (67, 8, 2, 64, "rms", 32, "halves"), (64, 16, 16, 128, "rms", 128, "pairs"), (301, 12, 4, 128, "unit", 96, "halves"),
    (33, 3, 3, 128, "fp32", 112, "pairs"), (2, 7, 7, 64, None, 16, "pairs"), (129, 32, 8, 128, "standard", 16, "halves"),
    (50, 6, 2, 64, "rms", 48, "pairs"), (9, 4, 4, 128, "standard", None, None), (5001, 16, 4, 128, "rms", 64, "pairs")])
def test_head_norm_rope(pa, dtype, rows, hq, hk, d, kind, rot, style):
    g = _gen(rows + d)
    fused = _randn(g, rows, hq + hk + 1, d, dtype=dtype, gain=2.0) + 0.25        # column ranges of one matrix, non-zero mean
    q, k = fused[:, :hq], fused[:, hq:hq + hk]
    norm, (qw, kw, qb, kb) = _norm(pa, g, kind, d, dtype)
    rope = cos = sin = None
    if rot:
        rope, cos, sin = _tables(pa, rot, style)
    pos = torch.randint(0, 4096, (rows,), generator=g, device="cuda", dtype=torch.int32)
    before = fused.clone()
    q2, k2 = pa.head_norm_rope(q, k, positions=pos, rope=rope, norm=norm)
    assert torch.equal(before, fused)
    for x, y, w, b in ((q, q2, qw, qb), (k, k2, kw, kb)):
        want, slack = ref.heads(x, kind, w, b, 1e-5, cos, sin, style, pos)
        _within(y, want, ref.heads_bound(want, slack, dtype), (rows, hq, hk))
    # one of the two alone, and in place, give the same bits
    only, none = pa.head_norm_rope(q, None, positions=pos, rope=rope, norm=norm)
    assert none is None and torch.equal(only, q2)
    none, only = pa.head_norm_rope(None, k, positions=pos, rope=rope, norm=norm)
    assert none is None and torch.equal(only, k2)
    pa.head_norm_rope(q, k, positions=pos, rope=rope, norm=norm, q_out=q, k_out=k)
    assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(fused[:, hq + hk:], before[:, hq + hk:])


def test_head_norm_rope_padding_and_far_positions(pa):
    g = _gen(5)
    q = _randn(g, 6, 2, 64, dtype=BF16)
    rope, cos, sin = _tables(pa, 64, "pairs", n=10)
    pos = _int([0, -1, 9, 10, -2**31, 2**31 - 1])
    out = torch.full_like(q, 7.0)
    pa.head_norm_rope(q, None, positions=pos, rope=rope, q_out=out)
    want, slack = ref.heads(q, None, None, None, 0, cos, sin, "pairs", pos)
    for r in (0, 2):
        _within(out[r], want[r], ref.heads_bound(want[r], slack[r], BF16))
    assert (out[[1, 4]] == 7).all()                       # padding: left as it was
    assert torch.isnan(out[[3, 5]]).all()                 # no angle known


def test_head_norm_of_extreme_values(pa):
    """A head of zeros stays zero (eps), a constant head has no deviation, a value of 1e15 does not overflow the fp32 sums."""
    q = torch.zeros(3, 1, 128, device="cuda")
    q[1] = 5.0
    q[2, 0, 3] = 1e15
    w = torch.ones(128, device="cuda")
    got, _ = pa.head_norm_rope(q, None, norm=pa.HeadNorm("rms", w))
    want, slack = ref.heads(q, "rms", w, None, 1e-5, None, None, None, None)
    _within(got, want, ref.heads_bound(want, slack, F32))
    got, _ = pa.head_norm_rope(q, None, norm=pa.HeadNorm("standard", w))
    assert (got[:2] == 0).all()
    got, _ = pa.head_norm_rope(q[:0], None, norm=pa.HeadNorm("rms", w))
    assert got.shape == (0, 1, 128)


# ---- batches ----------------------------------------------------------------------------------------------------------------
class Batch:
    """A pool with the pages of ragged sequences in random order; unused pages and places hold NaN."""

    def __init__(self, g, qs, past, hk, d, ps, dtype, extra_pages=3, spare=1, fill=math.nan):
        self.qs, self.past, self.ps = qs, past, ps
        self.lens = [a + b for a, b in zip(qs, past)]
        counts = [-(-n // ps) for n in self.lens]
        self.n_pages = sum(counts) + extra_pages
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        self.free = perm[sum(counts):]
        self.table = torch.full((len(qs), max(counts + [1]) + spare), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = perm[at:at + c]
            at += c
        self.k = torch.full((self.n_pages, hk, ps, d), fill, dtype=dtype, device="cuda")
        self.v = torch.full_like(self.k, fill)
        for b, n in enumerate(self.lens):
            for p in range(counts[b]):
                c = min(ps, n - p * ps)
                self.k[int(self.table[b, p]), :, :c] = _randn(g, hk, c, d, dtype=dtype, gain=1.5)
                self.v[int(self.table[b, p]), :, :c] = _randn(g, hk, c, d, dtype=dtype)
        self.starts = [0]
        for n in qs:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1]

    def make(self, pa, with_starts=True, max_keys="exact"):
        pages = pa.KVPages(self.k, self.v)
        batch = pa.PagedBatch(self.table, _int(self.lens), _int(self.starts) if with_starts else None, max_q=max(self.qs + [1]) if with_starts else 1,
                              max_keys=max(1, max(self.lens)) if max_keys == "exact" else max_keys)
        return pages, batch


APPENDS = [
    # qs, past, hq, hk, d, page, kind, rot, style, starts
    ([1], [0], 1, 1, 128, 16, None, 128, "pairs", False),
    ([1] * 64, [8 + (i * 37) % 128 for i in range(64)], 16, 16, 128, 16, None, 128, "pairs", False),
    ([1] * 5, [15, 16, 17, 31, 127], 8, 2, 64, 32, "rms", 64, "halves", True),
    ([0, 3, 0, 0, 40, 1, 0, 17, 0], [4, 0, 0, 9, 50, 100, 3, 63, 0], 6, 3, 128, 64, "standard", 48, "halves", True),
    ([200, 1, 333], [0, 700, 11], 32, 8, 128, 128, "rms", 128, "pairs", True),
    ([7], [300], 5, 5, 64, 256, "unit", 16, "pairs", True),
    ([2, 2], [0, 5], 2, 1, 128, 16, "fp32", None, None, True),
    ([1, 0] * 150, [3] * 300, 4, 2, 64, 16, "rms", 64, "pairs", True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_paged_append(pa, dtype, case):
    qs, past, hq, hk, d, ps, kind, rot, style, with_starts = APPENDS[case]
    g = _gen(case)
    b = Batch(g, qs, past, hk, d, ps, dtype)
    pages, batch = b.make(pa, with_starts)
    behind = 3 if with_starts else 0                               # rows behind the last sequence
    fused = _randn(g, b.rows + behind, hq + 2 * hk, d, dtype=dtype, gain=1.3)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
    norm, (qw, kw, qb, kb) = _norm(pa, g, kind, d, dtype)
    rope = cos = sin = None
    if rot:
        rope, cos, sin = _tables(pa, rot, style)
    at = torch.cat([torch.arange(p, p + n, device="cuda", dtype=torch.int32) for n, p in zip(qs, past)])
    given = torch.randint(0, 4096, (b.rows + behind,), generator=g, device="cuda", dtype=torch.int32)
    for positions in (None, given):
        b2k, b2v = b.k.clone(), b.v.clone()
        pos = at if positions is None else positions[:b.rows]
        want_k, slack_k = ref.heads(k[:b.rows], kind, kw, kb, 1e-5, cos, sin, style, pos)
        want_q, slack_q = ref.heads(q[:b.rows], kind, qw, qb, 1e-5, cos, sin, style, pos)
        q_out = torch.full((b.rows + behind, hq, d), 3.0, dtype=dtype, device="cuda")
        assert pa.paged_append(pages, batch, k, v, q=q, positions=positions, rope=rope, norm=norm, q_out=q_out) is q_out
        _within(q_out[:b.rows], want_q, ref.heads_bound(want_q, slack_q, dtype))
        assert (q_out[b.rows:] == 3).all()
        seq = [i for i, n in enumerate(qs) for _ in range(n)]
        page = b.table[seq, (at // ps).long()].long()
        off = (at % ps).long()
        _within(b.k[page, :, off], want_k, ref.heads_bound(want_k, slack_k, dtype))
        assert torch.equal(b.v[page, :, off], v[:b.rows])
        # every other place of the pool keeps its bits
        b2k[page, :, off], b2v[page, :, off] = b.k[page, :, off], b.v[page, :, off]
        assert torch.equal(b2k.nan_to_num(9), b.k.nan_to_num(9)) and torch.equal(b2v.nan_to_num(9), b.v.nan_to_num(9))
        # without queries: the same pages
        assert pa.paged_append(pages, batch, k, v, positions=positions, rope=rope, norm=norm) is None
        assert torch.equal(b2k.nan_to_num(9), b.k.nan_to_num(9)) and torch.equal(b2v.nan_to_num(9), b.v.nan_to_num(9))


def test_paged_append_skips(pa):
    """Bad page ids, rows before a sequence's beginning, rows beyond the table, negative positions, starts that lie outside the
    rows: nothing else is written."""
    g = _gen(1)
    ps, hk, d = 16, 2, 64
    k_pages = torch.full((4, hk, ps, d), 5.0, device="cuda")
    v_pages = torch.full_like(k_pages, 6.0)
    pages = pa.KVPages(k_pages, v_pages)
    table = _int([[0, 4], [-1, 1], [2**31 - 1, -2**31], [2, 3]])
    #            page 1 of seq 0 is bad; seq 1 wants page 0 (bad); seq 2 all bad; seq 3 has 3 rows but 2 positions
    lens, starts = _int([18, 3, 5, 2]), _int([0, 3, 5, 6, 9])
    x = _randn(g, 12, hk, d)
    q_out = torch.full((12, hk, d), 8.0, device="cuda")
    pos = _int([0] * 8 + [-1] + [0] * 3)                          # the second written row of seq 3 is padding
    pa.paged_append(pages, pa.PagedBatch(table, lens, starts, max_q=3), x, x, q=x, positions=pos, q_out=q_out)
    want_k, want_v = torch.full_like(k_pages, 5.0), torch.full_like(v_pages, 6.0)
    want_k[0, :, 15] = want_v[0, :, 15] = x[0]                    # position 15 of seq 0: the last of its good page
    want_k[2, :, 0] = want_v[2, :, 0] = x[7]                      # row 6 lies before the beginning of seq 3
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)
    assert torch.equal(q_out[:6], x[:6]) and torch.equal(q_out[7], x[7]) and (q_out[[6, 8, 9, 10, 11]] == 8).all()
    # lengths far outside the table and starts outside the rows
    k_pages.fill_(5.0), v_pages.fill_(6.0)
    pa.paged_append(pages, pa.PagedBatch(_int([[0], [1]]), _int([2**31 - 1, -7]), _int([-3, 2, 2**31 - 1]), max_q=3), x, x)
    assert torch.equal(k_pages[0, :, 14:16].transpose(0, 1), x[:2])
    assert (k_pages[0, :, :14] == 5).all() and (k_pages[1:] == 5).all() and (v_pages[1:] == 6).all()


# ---- attention ------------------------------------------------------------------------------------------------------------
ATTENDS = [
    # qs, past, hq, hk, d, page, starts
    ([1], [0], 1, 1, 128, 16, False),
    ([1], [136], 16, 16, 128, 16, False),
    ([1] * 9, [0, 1, 14, 15, 16, 30, 31, 32, 33], 4, 4, 128, 16, False),
    ([1] * 7, [62, 63, 64, 65, 127, 128, 1000], 8, 2, 64, 64, False),
    ([1] * 3, [2500, 17, 911], 16, 1, 128, 32, False),
    ([1] * 2, [40, 700], 24, 1, 128, 16, True),
    ([1, 0, 3, 5, 0, 2], [0, 9, 0, 30, 0, 100], 8, 2, 128, 16, True),
    ([4, 4, 4, 4], [28, 60, 0, 300], 4, 4, 128, 32, True),
    ([33, 1, 100, 7], [0, 64, 200, 31], 6, 3, 64, 16, True),
    ([129, 65], [0, 63], 4, 2, 128, 64, True),
    ([300], [5], 5, 5, 128, 128, True),
    ([2, 90], [1500, 3], 32, 8, 128, 256, True),
    ([17, 16, 15], [15, 16, 17], 3, 1, 64, 16, True),
    # more short parts than the chip has places: a wave for each
    ([1] * 64, [(i * 41) % 256 for i in range(64)], 16, 16, 128, 32, False),
    ([i % 4 for i in range(128)], [(i * 29) % 200 for i in range(128)], 8, 8, 64, 16, True),
    ([3] * 65, [0] * 65, 16, 16, 128, 16, True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_paged_attention(pa, dtype, causal, case):
    qs, past, hq, hk, d, ps, with_starts = ATTENDS[case]
    g = _gen(100 + case)
    b = Batch(g, qs, past, hk, d, ps, dtype)
    pages, batch = b.make(pa, with_starts)
    behind = 2 if with_starts else 0
    wide = _randn(g, b.rows + behind, hq + 1, d, dtype=dtype, gain=1.5)
    q = wide[:, 1:]                                                # strided rows
    out = torch.full((b.rows + behind, hq, d), 4.0, dtype=dtype, device="cuda")
    scale = d ** -0.5 if case % 2 else 0.21
    assert pa.paged_attention(q, pages, batch, causal=causal, scale=scale, out=out) is out
    want, bound, owned = ref.paged(q, b.k, b.v, b.table, b.lens, b.starts, causal, scale)
    _within(out[owned], want[owned], ref.attend_bound(want, bound, dtype)[owned], case)
    assert (out[~owned] == 4).all()
    # how the work is split may change the last bits, not the result: bounds far above the real lengths
    batch = pa.PagedBatch(b.table, _int(b.lens), _int(b.starts), max_q=1 + 3 * max(qs))
    again = pa.paged_attention(q[:b.rows], pages, batch, causal=causal, scale=scale)
    _within(again[owned[:b.rows]], want[owned], ref.attend_bound(want, bound, dtype)[owned], case)
    # a max_q that is too small costs time only
    again = pa.paged_attention(q[:b.rows], pages, pa.PagedBatch(b.table, _int(b.lens), _int(b.starts), max_q=1), causal=causal, scale=scale)
    _within(again[owned[:b.rows]], want[owned], ref.attend_bound(want, bound, dtype)[owned], case)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hq,hk", [(4, 4), (16, 2)])
def test_paged_attention_long(pa, dtype, hq, hk):
    """Tens of thousands of keys, split over many workgroups; one short sequence beside the long ones."""
    g = _gen(7)
    b = Batch(g, [1, 1, 1], [40000, 99, 70001], hk, 128, 128, dtype)
    pages, batch = b.make(pa, False)
    q = _randn(g, 3, hq, 128, dtype=dtype, gain=1.5)
    out = pa.paged_attention(q, pages, batch)
    want, bound, _ = ref.paged(q, b.k, b.v, b.table, b.lens, None, True, 128 ** -0.5)
    _within(out, want, ref.attend_bound(want, bound, dtype))
    assert torch.equal(out, pa.paged_attention(q, pages, batch))           # no atomics: the same bits again


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 5, 70])
def test_paged_attention_empty_rows_and_bad_pages(pa, dtype, n):
    """Rows that see no key give zeros: a sequence of length 0 or shorter than its rows, one whose pages are all bad.  A bad page in
    the middle is left out."""
    g = _gen(n)
    hq, hk, d, ps = 8, 2, 128, 16
    b = Batch(g, [n, n, n, n], [0, 120, 0, 200], hk, d, ps, dtype, spare=0)
    b.lens[0], b.lens[2] = 0, n // 2
    b.table[1, 2], b.table[1, 5], b.table[3, :] = -1, b.n_pages, -5
    pages, batch = b.make(pa)
    q = _randn(g, b.rows, hq, d, dtype=dtype, gain=1.5)
    for causal in (True, False):
        out = pa.paged_attention(q, pages, batch, causal=causal)
        want, bound, _ = ref.paged(q, b.k, b.v, b.table, b.lens, b.starts, causal, d ** -0.5)
        _within(out, want, ref.attend_bound(want, bound, dtype))
        assert (out[:n] == 0).all() and (out[3 * n:] == 0).all()
        if causal:
            assert (out[2 * n:2 * n + n - n // 2] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hq", [2, 8])
@pytest.mark.parametrize("n", [6, 150])
def test_paged_attention_masked_nan(pa, dtype, hq, n):
    """A NaN or an infinity in a key or value reaches exactly the rows that see it."""
    g = _gen(3)
    hk, d, ps = 2, 64, 16
    b = Batch(g, [n], [37], hk, d, ps, dtype)
    pages, batch = b.make(pa)
    q = _randn(g, n, hq, d, dtype=dtype)
    clean = pa.paged_attention(q, pages, batch)
    for pool, value in ((b.v, math.nan), (b.k, math.nan), (b.v, math.inf), (b.v, -math.inf)):
        for at in (37 + n - 1, 37 + n // 2, 37 + 1):
            page, off = int(b.table[0, at // ps]), at % ps
            kept = pool[page, 0, off].clone()
            pool[page, 0, off, 5] = value
            out = pa.paged_attention(q, pages, batch)
            pool[page, 0, off] = kept
            sees = torch.arange(n, device="cuda") + 37 >= at
            h = hq // hk                                           # key head 0 alone is touched
            assert torch.equal(out[:, h:], clean[:, h:]) and torch.equal(out[~sees], clean[~sees])
            hit = out[sees][:, :h]
            if pool is b.k:
                assert torch.isnan(hit).all()
            else:
                assert torch.equal(hit[..., :5], clean[sees][:, :h, :5]) and torch.equal(hit[..., 6:], clean[sees][:, :h, 6:])
                assert (torch.isnan(hit[..., 5]) if math.isnan(value) else hit[..., 5] == value).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 40])
def test_paged_attention_extreme_scores(pa, dtype, n):
    """Scores of +-1e4, equal scores of the lowest kind, and one key that outweighs all others."""
    d, ps = 64, 16
    k = torch.zeros(4, 1, ps, d, dtype=dtype, device="cuda")
    v = torch.randn(4, 1, ps, d, device="cuda").to(dtype)
    q = torch.zeros(n, 1, d, dtype=dtype, device="cuda")
    q[:, :, 0] = 128.0
    table = _int([[2, 0, 3]])
    pages, batch = pa.KVPages(k, v), pa.PagedBatch(table, _int([45]), _int([0, n]), max_q=n)
    for level in (-1e4, 1e4, -3e38, 3e38):
        k[..., 0] = level / 128.0
        out = pa.paged_attention(q, pages, batch, causal=False, scale=1.0)
        want, bound, _ = ref.paged(q, k, v, table, [45], [0, n], False, 1.0)
        # equal keys give equal scores bit for bit: their common size adds nothing to the bound of the weights
        flat = ref.half_step(dtype) * 2 + 128 * ref.U32
        _within(out, want, ref.attend_bound(want, flat * v.double().abs().max().expand_as(want), dtype))
    k[..., 0] = 0
    k[0, 0, 3, 0] = 100.0                                          # position 16 + 3
    out = pa.paged_attention(q, pages, batch, causal=False, scale=1.0)
    assert torch.equal(out, v[0, 0, 3].expand_as(out))


def test_paged_attention_beyond_32_bit_offsets(pa):
    """A pool of more than 2^31 values: appended to and read at its far end."""
    hk, ps, d = 8, 64, 128
    n_pages = (1 << 31) // (hk * ps * d) + 40
    k_pages = torch.empty(n_pages, hk, ps, d, dtype=BF16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    g = _gen(2)
    ids = list(range(n_pages - 5, n_pages))
    pages = pa.KVPages(k_pages, v_pages)
    x = _randn(g, 300, 3, hk, d, dtype=BF16)
    table, lens, starts = _int([ids]), _int([300]), _int([0, 300])
    pa.paged_append(pages, pa.PagedBatch(table, lens, starts, max_q=300), x[:, 0], x[:, 1])
    got = torch.cat([k_pages[i].transpose(0, 1) for i in ids])[:300]
    assert torch.equal(got, x[:, 0])
    for n in (300, 1):
        out = pa.paged_attention(x[300 - n:, 2], pages, pa.PagedBatch(table, lens, _int([0, n]), max_q=n))
        small_k, small_v = k_pages[ids[0]:].clone(), v_pages[ids[0]:].clone()
        want, bound, _ = ref.paged(x[300 - n:, 2], small_k, small_v, table - ids[0], [300], [0, n], True, d ** -0.5)
        _within(out, want, ref.attend_bound(want, bound, BF16))


# ---- shared prefixes ----------------------------------------------------------------------------------------------------------
SHARED = [
    # group sizes, sequences outside (before, behind), prefixes, queries, own past, hq, hk, d, page
    ([3], 0, 0, [50], [1] * 3, [0, 7, 30], 4, 4, 128, 16),
    ([20], 0, 0, [333], [1] * 20, [i * 3 for i in range(20)], 16, 16, 128, 64),
    ([5, 0, 2], 1, 2, [100, 70, 0], [1] * 10, [i * 11 for i in range(10)], 8, 2, 64, 16),
    ([4, 4], 0, 0, [1025, 17], [1, 3, 0, 5, 2, 2, 2, 2], [0] * 8, 6, 3, 128, 32),
    ([40, 30], 0, 0, [600, 2000], [1] * 70, [i % 50 for i in range(70)], 8, 2, 128, 128),
    ([2], 0, 1, [129], [60, 45, 3], [0, 10, 100], 4, 1, 64, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared_prefix_attention(pa, dtype, causal, case):
    sizes, before, behind, prefixes, qs, past, hq, hk, d, ps = SHARED[case]
    g = _gen(200 + case)
    n = len(qs)
    assert before + sum(sizes) + behind == n
    b = Batch(g, list(qs) + [0] * len(prefixes), list(past) + prefixes, hk, d, ps, dtype)     # prefixes as further sequences' pages
    pages = pa.KVPages(b.k, b.v)
    starts, lens = b.starts[:n + 1], b.lens[:n]
    table, prefix_table = b.table[:n].contiguous(), b.table[n:].contiguous()
    groups = [before]
    for s in sizes:
        groups.append(groups[-1] + s)
    batch = pa.PagedBatch(table, _int(lens), _int(starts), max_q=max(qs))
    prefix = pa.SharedPrefix(prefix_table, _int(prefixes), _int(groups), max_keys=max(prefixes))
    q = _randn(g, b.rows + 2, hq, d, dtype=dtype, gain=1.5)
    out = torch.full_like(q, 4.0)
    pa.shared_prefix_attention(q, pages, batch, prefix, causal=causal, out=out)
    want, bound, owned = ref.paged(q, b.k, b.v, table, lens, starts, causal, d ** -0.5, (prefix_table, prefixes, groups))
    _within(out[owned], want[owned], ref.attend_bound(want, bound, dtype)[owned], case)
    assert (out[~owned] == 4).all()
    if max(qs) == 1 and min(qs) == 1:
        batch = pa.PagedBatch(table, _int(lens), max_keys=max(lens))
        one = pa.shared_prefix_attention(q[:n], pages, batch, prefix, causal=causal)
        _within(one, want[:n], ref.attend_bound(want, bound, dtype)[:n], case)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_prefix_equals_one_long_sequence(pa, dtype):
    """A prefix shared by tables that repeat its pages gives what each sequence gives with the prefix as its own beginning; a prefix
    of bad pages or of no length leaves the own part alone."""
    g = _gen(9)
    hq, hk, d, ps, n = 8, 4, 128, 16, 12
    b = Batch(g, [1] * n + [0], [i * 5 for i in range(n)] + [320], hk, d, ps, dtype)
    pages = pa.KVPages(b.k, b.v)
    q = _randn(g, n, hq, d, dtype=dtype, gain=1.5)
    own, pre = b.table[:n].contiguous(), b.table[n:, :20].contiguous()
    lens = _int(b.lens[:n])
    batch = pa.PagedBatch(own, lens)
    got = pa.shared_prefix_attention(q, pages, batch, pa.SharedPrefix(pre, _int([320]), _int([0, n])))
    joined = torch.cat((pre.expand(n, -1), own), 1).contiguous()
    whole = pa.paged_attention(q, pages, pa.PagedBatch(joined, lens + 320))
    want, bound, _ = ref.paged(q, b.k, b.v, joined, [x + 320 for x in b.lens[:n]], None, True, d ** -0.5)
    for x in (got, whole):
        _within(x, want, ref.attend_bound(want, bound, dtype))
    want, bound, _ = ref.paged(q, b.k, b.v, own, b.lens[:n], None, True, d ** -0.5)
    for pre, length in ((torch.full_like(pre, -1), 320), (pre, 0), (pre, -4)):
        got = pa.shared_prefix_attention(q, pages, batch, pa.SharedPrefix(pre, _int([length]), _int([0, n])))
        _within(got, want, ref.attend_bound(want, bound, dtype))


# ---- together ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_run_of_steps(pa, dtype):
    """Prompts of ragged lengths, then single positions, through norm, rotation, append and attention; every step against the
    64-bit attention over all keys and values of the sequence so far.  Pages are handed out as the sequences grow."""
    g = _gen(11)
    hq, hk, d, ps, n = 8, 2, 128, 16, 4
    norm, (qw, kw, _, _) = _norm(pa, g, "rms", d, dtype)
    rope, cos, sin = _tables(pa, 128, "pairs")
    pages = pa.KVPages.create(40, ps, hk, d, dtype=dtype)
    pages.k.fill_(math.nan), pages.v.fill_(math.nan)
    table = torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    free = list(range(40))
    random.Random(0).shuffle(free)
    lens = [0] * n
    keys = [torch.zeros(0, hk, d, dtype=torch.float64, device="cuda") for _ in range(n)]
    vals = [x.clone() for x in keys]
    for step, qs in enumerate([[30, 1, 17, 64], [1] * 4, [1] * 4, [3, 0, 2, 1], [1] * 4]):
        for s in range(n):
            while -(-(lens[s] + qs[s]) // ps) > int((table[s] >= 0).sum()):
                table[s, int((table[s] >= 0).sum())] = free.pop()
            lens[s] += qs[s]
        starts = [sum(qs[:i]) for i in range(n + 1)]
        batch = pa.PagedBatch(table, _int(lens), _int(starts), max_q=max(qs), max_keys=max(lens))
        x = _randn(g, sum(qs), hq + 2 * hk, d, dtype=dtype)
        q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        q2 = pa.paged_append(pages, batch, k, v, q=q, rope=rope, norm=norm)
        pos = torch.cat([torch.arange(lens[s] - qs[s], lens[s], device="cuda", dtype=torch.int32) for s in range(n)])
        q3, k3 = pa.head_norm_rope(q, k, positions=pos, rope=rope, norm=norm)
        assert torch.equal(q2, q3)                                 # both entry points give the same bits
        out = pa.paged_attention(q2, pages, batch)
        for s in range(n):
            r = slice(starts[s], starts[s + 1])
            keys[s] = torch.cat((keys[s], k3[r].double()))
            vals[s] = torch.cat((vals[s], v[r].double()))
            if qs[s]:
                visible = torch.arange(lens[s] - qs[s] + 1, lens[s] + 1, device="cuda")
                there = torch.ones(lens[s], dtype=torch.bool, device="cuda")
                want, bound = ref.attend(q2[r], keys[s].transpose(0, 1), vals[s].transpose(0, 1), there, visible, d ** -0.5)
                _within(out[r], want, ref.attend_bound(want, bound, dtype), (step, s))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_steps(pa, dtype):
    """Append, attention and shared-prefix attention captured in two graphs, replayed in turn on changing contents with eager work
    between: every replay gives the eager bits."""
    g = _gen(12)
    hq, hk, d, ps, n = 16, 4, 128, 16, 6
    b = Batch(g, [1] * n + [0], [300, 20, 0, 77, 145, 1000] + [600], hk, d, ps, dtype, fill=0.0)
    pages = pa.KVPages(b.k, b.v)
    table, lens = b.table[:n].contiguous(), _int(b.lens[:n])
    batch = pa.PagedBatch(table, lens)
    prefix = pa.SharedPrefix(b.table[n:].contiguous(), _int([600]), _int([0, n]))
    rope, _, _ = _tables(pa, 128, "pairs")
    x = _randn(g, n, hq + 2 * hk, d, dtype=dtype)

    def step():
        q = pa.paged_append(pages, batch, x[:, hq:hq + hk], x[:, hq + hk:], q=x[:, :hq], rope=rope)
        return q, pa.paged_attention(q, pages, batch), pa.shared_prefix_attention(q, pages, batch, prefix)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(6):
        x.copy_(_randn(g, n, hq + 2 * hk, d, dtype=dtype))
        lens.copy_(_int([max(1, v - 13 * i) for v in b.lens[:n]]))
        graph, outs = graphs[i % 2]
        for o in outs:
            o.zero_()
        graph.replay()
        got = [o.clone() for o in outs] + [b.k.clone(), b.v.clone()]
        want = list(step()) + [b.k, b.v]
        for a, e in zip(got, want):
            assert torch.equal(a, e), i


def test_empty_batches(pa):
    """No rows, no sequences, rows of no sequence: nothing is written."""
    pages = pa.KVPages.create(2, 16, 2, 64, dtype=F32)
    pages.k.fill_(1.0), pages.v.fill_(2.0)
    x = torch.ones(3, 2, 64, device="cuda")
    out = torch.full_like(x, 5.0)
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    nobody = pa.PagedBatch(none, _int([]), _int([0]), max_q=1)
    assert (pa.paged_attention(x, pages, nobody, out=out) == 5).all()
    assert (pa.paged_append(pages, nobody, x, x, q=x, q_out=out) == 5).all()
    owned_by_none = pa.PagedBatch(_int([[0]]), _int([4]), _int([0, 0]), max_q=1)
    assert (pa.paged_attention(x, pages, owned_by_none, out=out) == 5).all()
    assert (pa.paged_append(pages, owned_by_none, x, x, q=x, q_out=out) == 5).all()
    prefix = pa.SharedPrefix(_int([[1]]), _int([16]), _int([0, 1]))
    assert (pa.shared_prefix_attention(x, pages, owned_by_none, prefix, out=out) == 5).all()
    assert pa.paged_attention(x[:0], pages, pa.PagedBatch(none, _int([]))).shape == (0, 2, 64)
    assert (pages.k == 1).all() and (pages.v == 2).all()


def test_one_batch_over_two_page_sizes(pa):
    """The bound of the lengths follows the pool that a call names, not the one that was used first."""
    x = torch.randn(1, 1, 64, device="cuda")
    batch = pa.PagedBatch(_int([[0]]), _int([40]))
    outs = []
    for ps in (16, 64, 16):
        k = torch.randn(1, 1, ps, 64, device="cuda", generator=_gen(ps))
        out = pa.paged_attention(x, pa.KVPages(k, k), batch)
        want, bound, _ = ref.paged(x, k, k, _int([[0]]), [40], None, True, 0.125)
        _within(out, want, ref.attend_bound(want, bound, F32))
        outs.append(out)
    assert torch.equal(outs[0], outs[2])


def test_other_streams(pa):
    """Two side streams at once, each with its own batch, give what the default stream gives."""
    g = _gen(13)
    made = []
    for i in range(2):
        b = Batch(g, [1] * 8, [700 + 211 * i] * 8, 4, 128, 64, BF16)
        pages, batch = b.make(pa, False)
        q = _randn(g, 8, 16, 128, dtype=BF16)
        made.append((q, pages, batch, pa.paged_attention(q, pages, batch)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        outs = []
        for s, (q, pages, batch, _) in zip(streams, made):
            with torch.cuda.stream(s):
                outs.append(pa.paged_attention(q, pages, batch))
        torch.cuda.synchronize()
        for o, (_, _, _, want) in zip(outs, made):
            assert torch.equal(o, want)


def test_python_layer_refusals(pa):
    q = torch.zeros(4, 4, 128, device="cuda", dtype=BF16)
    pages = pa.KVPages.create(2, 16, 2, 128)
    batch = pa.PagedBatch(_int([[0]] * 4), _int([1] * 4))
    prefix = pa.SharedPrefix(_int([[1]]), _int([3]), _int([0, 4]))
    kv = torch.zeros(4, 2, 128, device="cuda", dtype=BF16)
    rope = pa.RotaryTable.create(8, 128)
    norm = pa.HeadNorm("rms", torch.ones(128, device="cuda", dtype=BF16), torch.ones(128, device="cuda", dtype=BF16))
    refused = [
        lambda: pa.paged_attention(q.float(), pages, batch), lambda: pa.paged_attention(q[:3], pages, batch),
        lambda: pa.paged_attention(q[..., :64], pages, batch), lambda: pa.paged_attention(q[0], pages, batch),
        lambda: pa.paged_attention(q, pages, batch, out=q[:2]), lambda: pa.paged_attention(q, pages, batch, out=torch.zeros_like(q).transpose(0, 1)),
        lambda: pa.paged_attention(q.transpose(1, 2), pages, batch), lambda: pa.paged_append(pages, batch, kv, kv[:, :1]),
        lambda: pa.paged_append(pages, batch, kv.float(), kv.float()), lambda: pa.paged_append(pages, batch, kv, kv, q_out=q),
        lambda: pa.paged_append(pages, batch, q, q), lambda: pa.paged_append(pages, batch, kv, kv, positions=_int([0])),
        lambda: pa.paged_append(pages, batch, kv, kv, positions=torch.zeros(4, device="cuda", dtype=torch.int64)),
        lambda: pa.head_norm_rope(q, kv, rope=rope), lambda: pa.head_norm_rope(q, kv[:2]), lambda: pa.head_norm_rope(q.float(), None, norm=norm),
        lambda: pa.head_norm_rope(q, None, k_out=kv), lambda: pa.head_norm_rope(q, None, q_out=kv),
        lambda: pa.PagedBatch(_int([[0]] * 4), _int([1] * 3)), lambda: pa.PagedBatch(_int([[0]] * 4).long(), _int([1] * 4)),
        lambda: pa.PagedBatch(_int([[0]] * 4), _int([1] * 4), _int([0, 1])), lambda: pa.PagedBatch(_int([[0]] * 4), _int([1] * 4), max_q=2),
        lambda: pa.PagedBatch(_int([[0]] * 4), _int([1] * 4), _int([0] * 5), max_q=0),
        lambda: pa.paged_attention(q, pages, pa.PagedBatch(_int([[0]] * 4), _int([1] * 4), max_keys=17)),
        lambda: pa.shared_prefix_attention(q, pages, batch, pa.SharedPrefix(_int([[1]]), _int([3]), _int([0, 4]), max_keys=17)),
        lambda: pa.SharedPrefix(_int([[1]]), _int([3, 4]), _int([0, 4])), lambda: pa.SharedPrefix(_int([[1]]), _int([3]), _int([4])),
        lambda: pa.RotaryTable(rope.cos, rope.sin, style="other"), lambda: pa.RotaryTable(rope.cos.half(), rope.sin.half()),
        lambda: pa.KVPages(pages.k, pages.v.float()), lambda: pa.KVPages(pages.k, pages.v[:1]),
        lambda: pa.KVPages(pages.k.half(), pages.v.half())]
    for i, f in enumerate(refused):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    for f in (lambda: pa.paged_attention(q[:, :3], pages, batch), lambda: pa.paged_attention(q, pages, batch, scale=-1.0),
              lambda: pa.head_norm_rope(q, None, norm=pa.HeadNorm("rms")), lambda: pa.shared_prefix_attention(q, pages, batch, prefix, scale=0.0)):
        with pytest.raises(RuntimeError, match="lcmhip error -1"):
            f()
    x = q.clone().requires_grad_()
    for f in (lambda: pa.paged_attention(x, pages, batch), lambda: pa.head_norm_rope(x, None), lambda: pa.shared_prefix_attention(x, pages, batch, prefix)):
        with pytest.raises(RuntimeError, match="no backward"):
            f()
    with torch.no_grad():
        pa.paged_append(pages, batch, kv, kv)
        pa.paged_attention(x, pages, batch)
