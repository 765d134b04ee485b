"""Calls at the edges of what the paged cache operators (lcm.nn.paged_attention) document, against plain 64-bit statements."""

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


# ---- sequences longer than the cache can hold ---------------------------------------------------------------------------
def _overlong(pa, g, dtype, qs, lens, pages_each, ps, hk, d, max_keys):
    n, rows = len(qs), sum(qs)
    k, v = _randn(g, n * pages_each, hk, ps, d, dtype=dtype), _randn(g, n * pages_each, hk, ps, d, dtype=dtype)
    table = torch.randperm(n * pages_each, generator=g, device="cuda").to(torch.int32).view(n, pages_each)
    starts = [sum(qs[:i]) for i in range(n + 1)]
    batch = pa.PagedBatch(table, _int(lens), _int(starts), max_q=max(qs), max_keys=max_keys)
    bound = pages_each * ps if max_keys is None else max_keys
    return pa.KVPages(k, v), batch, table, starts, rows, bound


OVERLONG = [
    # qs, lens, pages of a sequence, page size, max_keys
    ([1, 1, 1], [16, 17, 2**31 - 1], 1, 16, None),
    ([4, 4, 4, 4], [18, 20, 24, 21], 4, 16, 20),             # the table has room behind max_keys
    ([3, 150, 70], [2**31 - 1, 140, 200], 4, 32, 127),
    ([2, 3], [300, 33], 2, 16, 31)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", range(len(OVERLONG)))
def test_positions_past_the_bound_are_not_there(pa, dtype, case):
    """Row t of a sequence is position len - (end - t) however long the sequence is; a position from max_keys on has no place:
    nothing is stored over the positions before it, its row is skipped, and rows see the keys below max_keys only."""
    qs, lens, each, ps, max_keys = OVERLONG[case]
    g = _gen(300 + case)
    hq, hk, d = 4, 2, 64
    pages, batch, table, starts, rows, bound = _overlong(pa, g, dtype, qs, lens, each, ps, hk, d, max_keys)
    rope = pa.RotaryTable.create(256, d)
    x = _randn(g, rows, hq + 2 * hk, d, dtype=dtype)
    q_out = torch.full((rows, hq, d), 3.0, dtype=dtype, device="cuda")
    want_k, want_v = pages.k.double(), pages.v.double()
    bound_k = torch.zeros_like(want_k)
    at = [lens[b] - (starts[b + 1] - t) for b in range(len(qs)) for t in range(starts[b], starts[b + 1])]
    seq = [b for b, n in enumerate(qs) for _ in range(n)]
    stored = [t for t in range(rows) if 0 <= at[t] < bound]
    pos = _int([max(0, min(c, 255)) for c in at])
    y, slack = ref.heads(x[:, hq:hq + hk], None, None, None, 0, rope.cos, rope.sin, "pairs", pos)
    for t in stored:
        page, off = int(table[seq[t], at[t] // ps]), at[t] % ps
        want_k[page, :, off], want_v[page, :, off] = y[t], x[t, hq + hk:].double()
        bound_k[page, :, off] = ref.heads_bound(y[t], slack[t], dtype)
    pa.paged_append(pages, batch, x[:, hq:hq + hk], x[:, hq + hk:], q=x[:, :hq], rope=rope, q_out=q_out)
    _within(pages.k, want_k, bound_k, "keys")
    assert torch.equal(pages.v.double(), want_v)
    y, slack = ref.heads(x[:, :hq], None, None, None, 0, rope.cos, rope.sin, "pairs", pos)
    skipped = [t for t in range(rows) if t not in stored]
    assert (q_out[skipped] == 3).all()
    _within(q_out[stored], y[stored], ref.heads_bound(y, slack, dtype)[stored], "queries")
    # what the rows see: positions up to their own, and none from the bound on
    q = x[:, :hq].contiguous()
    for causal in (True, False):
        out = pa.paged_attention(q, pages, batch, causal=causal)
        for b in range(len(qs)):
            r = slice(starts[b], starts[b + 1])
            keys = min(lens[b], bound)
            kk, there = ref.gather(pages.k, table[b], keys, ps)
            vv, _ = ref.gather(pages.v, table[b], keys, ps)
            visible = torch.tensor([max(0, min(c + 1, keys)) if causal else keys for c in at[r]], device="cuda")
            want, slack = ref.attend(q[r], kk, vv, there, visible, d ** -0.5)
            _within(out[r], want, ref.attend_bound(want, slack, dtype), (causal, b))


def test_bad_places_are_skipped(pa):
    """Bad page ids, rows before a sequence's beginning and behind its table, negative positions, starts that lie outside the rows:
    nothing else is written."""
    g = _gen(1)
    ps, hk, d = 16, 2, 64
    k_pages = torch.full((4, hk, ps, d), 5.0, device="cuda")
    v_pages = torch.full_like(k_pages, 6.0)
    pages = pa.KVPages(k_pages, v_pages)
    table = _int([[0, 4], [-1, 1], [2**31 - 1, -2**31], [2, 3]])
    lens, starts = _int([18, 3, 5, 2]), _int([0, 3, 5, 6, 9])
    x = _randn(g, 12, hk, d)
    q_out = torch.full((12, hk, d), 8.0, device="cuda")
    pos = _int([0] * 8 + [-1] + [0] * 3)
    pa.paged_append(pages, pa.PagedBatch(table, lens, starts, max_q=3), x, x, q=x, positions=pos, q_out=q_out)
    want_k, want_v = torch.full_like(k_pages, 5.0), torch.full_like(v_pages, 6.0)
    want_k[0, :, 15] = want_v[0, :, 15] = x[0]
    want_k[2, :, 0] = want_v[2, :, 0] = x[7]
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)
    assert torch.equal(q_out[:6], x[:6]) and torch.equal(q_out[7], x[7]) and (q_out[[6, 8, 9, 10, 11]] == 8).all()
    # a length far behind the table and a negative one, starts outside the rows: no row has a place
    k_pages.fill_(5.0), v_pages.fill_(6.0)
    pa.paged_append(pages, pa.PagedBatch(_int([[0], [1]]), _int([2**31 - 1, -7]), _int([-3, 2, 2**31 - 1]), max_q=3), x, x)
    assert (k_pages == 5).all() and (v_pages == 6).all()
    # the same starts, with a length that gives the first range its places: its two rows that exist are the positions 14 and 15
    pa.paged_append(pages, pa.PagedBatch(_int([[0], [1]]), _int([16, -7]), _int([-3, 2, 2**31 - 1]), max_q=3), x, x)
    assert torch.equal(k_pages[0, :, 14:16].transpose(0, 1), x[:2]) and torch.equal(v_pages[0, :, 14:16].transpose(0, 1), x[:2])
    assert (k_pages[0, :, :14] == 5).all() and (k_pages[1:] == 5).all() and (v_pages[1:] == 6).all()


# ---- derivatives -------------------------------------------------------------------------------------------------------------
def test_every_tensor_of_a_call_is_refused_with_a_gradient_or_a_tangent(pa):
    """Nothing that a derivative would flow through is used without one: inputs, pages, norm weights and biases, rotary tables and
    outputs that the caller gives."""
    n, hq, hk, d, ps = 3, 4, 2, 64, 16
    g = _gen(17)

    def made(name, change):
        """The four calls on fresh tensors, the one called `name` passed through `change`."""
        t = dict(q=_randn(g, n, hq, d), k=_randn(g, n, hk, d), v=_randn(g, n, hk, d), k_pages=_randn(g, 4, hk, ps, d), v_pages=_randn(g, 4, hk, ps, d),
                 qw=torch.ones(d, device="cuda"), kw=torch.ones(d, device="cuda"), qb=torch.zeros(d, device="cuda"), kb=torch.zeros(d, device="cuda"),
                 cos=torch.ones(64, d // 2, device="cuda"), sin=torch.zeros(64, d // 2, device="cuda"), q_out=torch.zeros(n, hq, d, device="cuda"),
                 k_out=torch.zeros(n, hk, d, device="cuda"))
        if name:
            t[name] = change(t[name])
        pages = pa.KVPages(t["k_pages"], t["v_pages"])
        batch = pa.PagedBatch(_int([[0], [1], [2]]), _int([5, 6, 7]))
        prefix = pa.SharedPrefix(_int([[3]]), _int([9]), _int([0, 3]))
        how = dict(rope=pa.RotaryTable(t["cos"], t["sin"]), norm=pa.HeadNorm("standard", t["qw"], t["kw"], t["qb"], t["kb"]))
        pos = _int([4, 5, 6])
        heads, store = ["cos", "sin", "qw", "kw", "qb", "kb", "q", "k", "q_out"], ["k_pages", "v_pages", "v"]
        return [(heads + ["k_out"], lambda: pa.head_norm_rope(t["q"], t["k"], positions=pos, q_out=t["q_out"], k_out=t["k_out"], **how)),
                (heads + store, lambda: pa.paged_append(pages, batch, t["k"], t["v"], q=t["q"], q_out=t["q_out"], **how)),
                (["q", "q_out", "k_pages", "v_pages"], lambda: pa.paged_attention(t["q"], pages, batch, out=t["q_out"])),
                (["q", "q_out", "k_pages", "v_pages"], lambda: pa.shared_prefix_attention(t["q"], pages, batch, prefix, out=t["q_out"]))]

    for _, call in made(None, None):
        call()
    names = ["q", "k", "v", "k_pages", "v_pages", "qw", "kw", "qb", "kb", "cos", "sin", "q_out", "k_out"]
    for name in names:
        for uses, call in made(name, lambda x: x.requires_grad_()):
            if name in uses:
                with pytest.raises(RuntimeError, match="no backward"):
                    call()
                    pytest.fail(f"a gradient of {name} was lost")
            with torch.no_grad():
                call()
    with torch.autograd.forward_ad.dual_level():
        for _, call in made(None, None):
            call()
        for name in names:
            for uses, call in made(name, lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))):
                if name in uses:
                    with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode"):
                        call()
                        pytest.fail(f"a tangent of {name} was lost")
    # transforms of torch.func hand in tensors without storage
    pages, batch = pa.KVPages.create(1, 16, 2, 64, dtype=F32), pa.PagedBatch(_int([[0]] * n), _int([1] * n))
    q = _randn(g, n, hq, d)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: pa.paged_attention(x, pages, batch), (q,), (q,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: pa.paged_attention(x, pages, batch).sum())(q)


# ---- rows that are skipped -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_skipped_rows_between_others(pa, dtype):
    """Rows of no sequence, of negative positions and of missing pages, alone in a wave or beside rows that are stored: what they
    hold (NaN here) reaches nothing, their outputs stay, and their neighbours are as without them."""
    g = _gen(23)
    hq, hk, d, ps, rows = 5, 2, 64, 16, 77
    x = _randn(g, rows, hq + 2 * hk, d, dtype=dtype)
    starts, lens = [3, 20, 40, 70], [17, 30, 30]
    table = _int([[0, 1], [2, -1], [3, 4]])
    pos = _int([-1 if t % 3 == 0 else t for t in range(rows)])
    seq = [next((b for b in range(3) if starts[b] <= t < starts[b + 1]), -1) for t in range(rows)]
    at = [lens[seq[t]] - (starts[seq[t] + 1] - t) if seq[t] >= 0 else -1 for t in range(rows)]
    lives = [t for t in range(rows) if seq[t] >= 0 and t % 3 and at[t] >= 0]
    stored = [t for t in lives if int(table[seq[t], at[t] // ps]) >= 0]
    rope, norm = pa.RotaryTable.create(128, d, style="halves"), pa.HeadNorm("rms", torch.ones(d, device="cuda", dtype=dtype), torch.ones(d, device="cuda", dtype=dtype))
    x[[t for t in range(rows) if t not in lives]] = float("nan")
    pages = pa.KVPages(torch.full((5, hk, ps, d), 5.0, device="cuda", dtype=dtype), torch.full((5, hk, ps, d), 6.0, device="cuda", dtype=dtype))
    q_out = torch.full((rows, hq, d), 3.0, device="cuda", dtype=dtype)
    pa.paged_append(pages, pa.PagedBatch(table, _int(lens), _int(starts), max_q=30), x[:, hq:hq + hk], x[:, hq + hk:], q=x[:, :hq], positions=pos,
                    rope=rope, norm=norm, q_out=q_out)
    alone_q, alone_k = pa.head_norm_rope(x[lives][:, :hq], x[lives][:, hq:hq + hk], positions=pos[lives].contiguous(), rope=rope, norm=norm)
    want_q = torch.full_like(q_out, 3.0)
    want_q[lives] = alone_q
    assert torch.equal(q_out, want_q)
    want_k, want_v = torch.full_like(pages.k, 5.0), torch.full_like(pages.v, 6.0)
    for t in stored:
        page, off = int(table[seq[t], at[t] // ps]), at[t] % ps
        want_k[page, :, off], want_v[page, :, off] = alone_k[lives.index(t)], x[t, hq + hk:]
    assert torch.equal(pages.k, want_k) and torch.equal(pages.v, want_v)


# ---- precision and long lists ----------------------------------------------------------------------------------------------------
def _attend64(q, k, v, visible, scale, weight_error):
    """q (n, hq, d), k / v (hk, keys, d) in 64 bits, visible (n, keys) (every row sees one): the result in 64 bits and its bound in
    fp32 arithmetic whose weights are off by `weight_error` each."""
    n, hq, d = q.shape
    hk, keys, _ = k.shape
    x = q.double().view(n, hk, hq // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    mask = visible[None, None].expand(hk, hq // hk, n, keys).reshape(hk, -1, keys)
    s = (torch.bmm(x, k.transpose(1, 2).contiguous()) * scale).masked_fill(~mask, -torch.inf)
    p = torch.softmax(s, -1)
    out, spread = torch.bmm(p, v), torch.bmm(p, v.abs())
    # a score: d products and sums, the scaling to base 2 and the subtraction of the maximum; exp2 itself 2 steps
    size = torch.bmm(x.abs(), k.abs().transpose(1, 2).contiguous()).masked_fill(~mask, 0.0).amax(-1)
    top = s.masked_fill(~mask, 0.0).abs().amax(-1)
    ds = (d + 8) * ref.U32 * size * scale * 1.4427 + 4 * ref.U32 * top + 2 * ref.U32
    many = (64 + mask.sum(-1) / 16 + 1) * ref.U32
    bound = spread * (2 * ds + weight_error + 2 * many)[..., None]
    back = lambda t: t.view(hk, hq // hk, n, d).permute(2, 0, 1, 3).reshape(n, hq, d)
    return back(out), back(bound)


@pytest.mark.parametrize("past,hq,hk,d,ps", [(137, 16, 16, 128, 16), (3000, 16, 4, 64, 64), (20000, 8, 8, 128, 128), (260, 5, 5, 64, 32)])
def test_weights_of_few_rows_are_not_rounded_to_the_operand_type(pa, past, hq, hk, d, ps):
    """With few rows a list the matrix unit waits for memory, and a weight enters the second product as two bf16 numbers, its upper bits
    and the rest.  Cutting a weight to bf16 leaves less than a step, finfo(bf16).eps = 2^-7 of it; the rest is rounded, half_step(bf16) =
    2^-8 of itself: 2^-7 2^-8 = 2^-15 of the weight is lost at most, 2^-24 is added, and the output has its own rounding."""
    g = _gen(past)
    lens = [past, past // 2 + 1, 1]
    each = -(-past // ps)
    k, v = _randn(g, 3 * each, hk, ps, d, dtype=BF16, gain=1.5), _randn(g, 3 * each, hk, ps, d, dtype=BF16)
    table = torch.randperm(3 * each, generator=g, device="cuda").to(torch.int32).view(3, each)
    q = _randn(g, 3, hq, d, dtype=BF16, gain=0.5)
    out = pa.paged_attention(q, pa.KVPages(k, v), pa.PagedBatch(table, _int(lens)))
    for b in range(3):
        kk, _ = ref.gather(k, table[b], lens[b], ps)
        vv, _ = ref.gather(v, table[b], lens[b], ps)
        want, bound = _attend64(q[b:b + 1], kk, vv, torch.ones(1, lens[b], dtype=torch.bool, device="cuda"), d ** -0.5, 2.0 ** -15 + ref.U32)
        _within(out[b:b + 1], want, ref.attend_bound(want, bound, BF16), b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,past", [(1, 0), (1, 31), (1, 300), (3, 200), (40, 100)])
def test_an_infinite_value_that_every_row_sees(pa, dtype, n, past):
    """A value of +-inf under a weight that is not 0 gives +-inf in its dimension and nothing elsewhere, whatever the weight's low bits
    are; both signs together give NaN."""
    g = _gen(400 + n + past)
    hq, hk, d, ps = 4, 2, 64, 16
    each = -(-(past + n) // ps)
    k, v = _randn(g, each, hk, ps, d, dtype=dtype), _randn(g, each, hk, ps, d, dtype=dtype)
    table = torch.randperm(each, generator=g, device="cuda").to(torch.int32).view(1, each)
    pages, batch = pa.KVPages(k, v), pa.PagedBatch(table, _int([past + n]), _int([0, n]), max_q=n)
    q = _randn(g, n, hq, d, dtype=dtype, gain=0.5)
    clean = pa.paged_attention(q, pages, batch)
    for at in sorted({0, past // 3, past // 2, max(0, past - 1), past}):
        page, off = int(table[0, at // ps]), at % ps
        for head in range(hk):
            kept = v[page, head, off].clone()
            v[page, head, off, 7], v[page, head, off, 40] = float("inf"), -float("inf")
            out = pa.paged_attention(q, pages, batch)
            mine = torch.arange(hq, device="cuda") // (hq // hk) == head
            assert torch.equal(out[:, ~mine], clean[:, ~mine])
            hit, rest = out[:, mine], [x for x in range(d) if x not in (7, 40)]
            assert (hit[..., 7] == float("inf")).all() and (hit[..., 40] == -float("inf")).all(), (at, head)
            assert torch.equal(hit[..., rest], clean[:, mine][..., rest])
            if past:                                               # another key's infinity of the other sign
                other = (at + 1) % past if (at + 1) % past != at else 0
                opage, ooff = int(table[0, other // ps]), other % ps
                if (opage, ooff) != (page, off):
                    okept = v[opage, head, ooff].clone()
                    v[opage, head, ooff, 7] = -float("inf")
                    assert torch.isnan(pa.paged_attention(q, pages, batch)[:, mine, 7]).all()
                    v[opage, head, ooff] = okept
            v[page, head, off] = kept


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs,past,parts", [(32, (2000, 4000), 1), (16, (8000, 9000), 2)])
def test_parts_of_more_pages_than_a_wave_holds(pa, dtype, causal, seqs, past, parts):
    """Many rows against parts of more than 64 pages of 16: the page ids of a part are held 64 at a time.  Missing pages lie on both sides
    of every 64th and on it; the pool is NaN wherever no sequence has a page."""
    import ctypes as C
    from lcm import _hip
    g = _gen(seqs)
    r = torch.Generator().manual_seed(seqs)
    hq = hk = 8
    d, ps = 64, 16
    qs = [200 + int(torch.randint(0, 30, (1,), generator=r)) for _ in range(seqs)]
    lens = [q + int(torch.randint(past[0], past[1] + 1, (1,), generator=r)) for q in qs]
    counts = [-(-n // ps) for n in lens]
    ids = torch.randperm(sum(counts) + 50, generator=g, device="cuda").to(torch.int32)
    table = torch.full((seqs, max(counts)), -1, dtype=torch.int32, device="cuda")
    k = torch.full((sum(counts) + 50, hk, ps, d), float("nan"), dtype=dtype, device="cuda")
    v = torch.full_like(k, float("nan"))
    first = 0
    for b, c in enumerate(counts):
        mine = ids[first:first + c]
        first += c
        table[b, :c] = mine
        k[mine.long()], v[mine.long()] = _randn(g, c, hk, ps, d, dtype=dtype, gain=1.5), _randn(g, c, hk, ps, d, dtype=dtype)
    for b in range(seqs):                                              # a quarter of the sequences has all its pages
        if b % 4:
            for at in ([63, 64, 65, 128], [62, 127, 129], [64, 191, 192])[b % 4 - 1]:
                if at < counts[b]:
                    table[b, at] = (-1, k.shape[0], 2**31 - 1)[at % 3]
    starts = [sum(qs[:i]) for i in range(seqs + 1)]
    rows = starts[-1]
    q = _randn(g, rows, hq, d, dtype=dtype, gain=1.0)
    pages, batch = pa.KVPages(k, v), pa.PagedBatch(table, _int(lens), _int(starts), max_q=max(qs), max_keys=max(lens))
    size = C.c_size_t()
    _hip.check(_hip.lib.lcmhip_paged_attention_workspace(pages._ref, batch._bind(pages, rows), rows, hq, C.byref(size)))
    assert size.value == (0 if parts == 1 else parts * rows * hq * (4 * d + 8))       # the parts are as long as this test wants them
    out = pa.paged_attention(q, pages, batch, causal=causal)
    for b in range(seqs):
        kk, there = ref.gather(k, table[b], lens[b], ps)
        vv, _ = ref.gather(v, table[b], lens[b], ps)
        kk, vv = kk * 1, vv * 1
        kk[:, ~there], vv[:, ~there] = 0.0, 0.0
        visible = there[None].expand(qs[b], -1).clone()
        if causal:
            visible &= torch.arange(lens[b], device="cuda")[None] <= torch.arange(lens[b] - qs[b], lens[b], device="cuda")[:, None]
        mine = slice(starts[b], starts[b + 1])
        want, bound = _attend64(q[mine], kk, vv, visible, d ** -0.5, ref.half_step(dtype) if dtype is BF16 else 0.0)
        _within(out[mine], want, ref.attend_bound(want, bound, dtype), b)
