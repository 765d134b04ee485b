"""Timed cases of the paged key/value cache operators (`lcm.nn.paged_attention`) and their plain forms.

Four operators that a decoder stack calls between its q / k / v products and its output product:

  head_norm_rope            norm of every query and key head and the position rotation, one pass
  paged_append              keys and values into the pages of a cache, keys (and queries) normed and rotated on the way
  paged_attention           queries of a ragged batch over the pages of their sequences
  shared_prefix_attention   the same for groups of sequences that begin with one common prefix

`run` computes a case in its plain form, elementary torch operations in 32 bits, or with `own` set makes the calls of
the package.  `exact` states the same results once more in 64 bits.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of the 1.6B two-tower stack: 64 documents, 16 heads of 128
        dict(name="heads_decode", op="heads", dtype="bf16", rows=64, hq=16, hk=16, d=128, rot=128, style="pairs", norm="rms",
             max_pos=4096),
        # small heads, half of each rotated, LayerNorm with bias, slices of one fused product: fp32, an odd row count
        dict(name="heads_f32_odd", op="heads", dtype="f32", rows=1001, hq=8, hk=2, d=64, rot=32, style="halves", norm="standard",
             max_pos=4096),
        # prompts of a whole batch at once, grouped key heads
        dict(name="heads_prompts", op="heads", dtype="bf16", rows=16384, hq=32, hk=8, d=128, rot=128, style="halves", norm="rms",
             max_pos=4096),
        # one new sentence for each of 64 documents of 8 prompt + up to 128 generated sentences, rotated on the way
        dict(name="append_decode", op="append", dtype="bf16", seqs=64, q_lo=1, q_hi=1, past_lo=8, past_hi=135, page=16, hq=16, hk=16,
             d=128, rot=128, style="pairs", norm="none", max_pos=4096),
        # ragged prompts appended behind ragged histories, queries rotated in the same pass, norms included
        dict(name="append_prompts", op="append", dtype="bf16", seqs=37, q_lo=1, q_hi=777, past_lo=0, past_hi=1500, page=64, hq=32, hk=8,
             d=128, rot=128, style="pairs", norm="rms", max_pos=4096),
        # one document of 8 + 129 sentences, one query, fp32: nothing but latency
        dict(name="attend_small", op="attend", dtype="f32", seqs=1, q_lo=1, q_hi=1, past_lo=136, past_hi=136, page=16, hq=16, hk=16, d=128),
        # 64 documents near the context limit, one query each, every head its own keys
        dict(name="attend_docs", op="attend", dtype="bf16", seqs=64, q_lo=1, q_hi=1, past_lo=1000, past_hi=3799, page=64, hq=16, hk=16, d=128),
        # few rows, very long caches: the keys' axis is what there is to split
        dict(name="attend_long", op="attend", dtype="bf16", seqs=2, q_lo=1, q_hi=1, past_lo=120001, past_hi=131071, page=128, hq=32, hk=8, d=128),
        # prompts behind cached histories, causal
        dict(name="attend_prompts", op="attend", dtype="bf16", seqs=8, q_lo=1500, q_hi=2048, past_lo=0, past_hi=2048, page=64, hq=32, hk=8, d=128),
        # 64 continuations of one document
        dict(name="shared_docs", op="shared", dtype="bf16", groups=1, seqs=64, prefix_lo=3701, prefix_hi=3701, q_lo=1, q_hi=1, past_lo=0,
             past_hi=127, page=64, hq=16, hk=16, d=128),
        # a few fp32 rows over a short prefix, odd lengths, up to 5 queries a sequence
        dict(name="shared_f32_odd", op="shared", dtype="f32", groups=3, seqs=13, prefix_lo=301, prefix_hi=907, q_lo=1, q_hi=5, past_lo=0,
             past_hi=61, page=16, hq=8, hk=2, d=64),
        # four prompts of tens of thousands of positions, 48 answers to each
        dict(name="shared_long", op="shared", dtype="bf16", groups=4, seqs=192, prefix_lo=20000, prefix_hi=32768, q_lo=1, q_hi=1, past_lo=0,
             past_hi=1023, page=128, hq=32, hk=8, d=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    """One more case of the ranges above: rows, sequences and lengths spread over their logarithm, both types, head widths
    of 64 and 128, grouped and plain heads, page sizes of 16 to 256."""
    while True:
        op = rng.choice(["heads", "append", "attend", "attend", "shared", "shared"])
        hq, hk = rng.choice([(16, 16), (32, 8), (8, 2), (32, 32), (12, 4), (16, 1), (5, 5)])
        d = rng.choice([64, 128, 128])
        c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), hq=hq, hk=hk, d=d)
        if op in ("heads", "append"):
            c.update(rot=rng.choice([d, d, d // 2]), style=rng.choice(["pairs", "halves"]), norm=rng.choice(["none", "rms", "standard", "unit"]),
                     max_pos=rng.choice([4096, 32768]))
        if op == "heads":
            c.update(rows=_log(rng, 1, 16384))
        else:
            c.update(page=rng.choice([16, 32, 64, 128, 256]))
            if op == "append":
                q = rng.choice([1, _log(rng, 2, 1024)])
                c.update(seqs=_log(rng, 1, 256), q_lo=max(1, q // 3), q_hi=q, past_lo=0, past_hi=_log(rng, 1, 2000))
            elif op == "attend":
                q = rng.choice([1, 1, _log(rng, 2, 2048)])
                past = _log(rng, 16, 131072)
                c.update(seqs=_log(rng, 1, 256), q_lo=max(1, q // 2), q_hi=q, past_lo=past // rng.choice([1, 2, 8]), past_hi=past)
            else:
                q = rng.choice([1, 1, _log(rng, 2, 16)])
                prefix = _log(rng, 64, 32768)
                groups = rng.choice([1, 1, 2, 4])
                c.update(groups=groups, seqs=groups * _log(rng, 1, 64), prefix_lo=prefix // rng.choice([1, 2]), prefix_hi=prefix,
                         q_lo=max(1, q // 2), q_hi=q, past_lo=0, past_hi=_log(rng, 1, 1024))
        w = work(c)
        pool = 0 if op == "heads" else 2 * sum(_slots(c)) * hk * d
        if w["bytes"] <= 1.2e9 and w["flops"] <= 2e11 and pool <= 8e8:
            return c


def _spread(n, lo, hi, salt):
    r = random.Random(salt)
    return [r.randint(lo, hi) for _ in range(n)]


def _shape(case):
    """Host lists of a batch: queries, keys before them (a sequence's own), sequences of each group, prefix lengths."""
    n = case["seqs"]
    qs = _spread(n, case["q_lo"], case["q_hi"], 1)
    past = _spread(n, case["past_lo"], case["past_hi"], 2)
    if case["op"] != "shared":
        return qs, past, [n], [0]
    g = case["groups"]
    sizes = [n // g + (1 if i < n % g else 0) for i in range(g)]
    return qs, past, sizes, _spread(g, case["prefix_lo"], case["prefix_hi"], 3)


def _slots(case):
    """Positions that the pages of every sequence and of every prefix hold."""
    qs, past, _, prefix = _shape(case)
    ps = case["page"]
    return [-(-n // ps) * ps for n in [a + b for a, b in zip(qs, past)] + prefix]


def work(case):
    """Every input byte the result depends on once, every output byte once; products at two operations each."""
    size = 2 if case["dtype"] == "bf16" else 4
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "heads":
        rows = case["rows"]
        values = rows * (hq + hk) * d
        return {"bytes": 2 * values * size + rows * (4 + case["rot"] * 4), "flops": values * 8}
    qs, past, sizes, prefix = _shape(case)
    rows = sum(qs)
    if case["op"] == "append":
        values = rows * (hq + 2 * hk) * d
        return {"bytes": 2 * values * size + rows * case["rot"] * 4 + len(qs) * 12, "flops": rows * (hq + hk) * d * 8}
    keys = sum(q + p for q, p in zip(qs, past)) + sum(prefix)
    pairs = sum(q * p + q * (q + 1) // 2 for q, p in zip(qs, past))
    i = 0
    for n, length in zip(sizes, prefix):
        pairs += sum(qs[i:i + n]) * length
        i += n
    return {"bytes": 2 * rows * hq * d * size + 2 * keys * hk * d * size + 4 * (keys // case["page"] + len(qs)),
            "flops": 4 * pairs * hq * d}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    dev, dt = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    hq, hk, d = case["hq"], case["hk"], case["d"]

    def normal(*shape, gain=1.0):
        return (torch.randn(*shape, generator=g, device=dev, dtype=torch.float32) * gain).to(dt)

    s = {"case": case}
    if "rot" in case:
        half = case["rot"] // 2
        angle = torch.arange(case["max_pos"], device=dev, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)[None, :]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["norm"] in ("rms", "standard"):
            s["qw"], s["kw"] = 1 + normal(d, gain=0.1), 1 + normal(d, gain=0.1)
        if case["norm"] == "standard":
            s["qb"], s["kb"] = normal(d, gain=0.1), normal(d, gain=0.1)
    rows = case["rows"] if case["op"] == "heads" else sum(_shape(case)[0])
    # q, k and v as a stacked product leaves them: column ranges of one matrix
    if case["op"] in ("heads", "append"):
        fused = normal(rows, hq + 2 * hk, d, gain=1.7)
        s["q"], s["k"], s["v"] = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
        s["positions"] = torch.randint(0, case["max_pos"], (rows,), generator=g, device=dev, dtype=torch.int32)
    else:
        s["q"] = normal(rows, hq, d, gain=1.5)
    if case["op"] == "heads":
        return s
    qs, past, sizes, prefix = _shape(case)
    ps = case["page"]
    slots = _slots(case)
    n_pages = sum(slots) // ps + 1
    s["k_pages"], s["v_pages"] = normal(n_pages, hk, ps, d), normal(n_pages, hk, ps, d)
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    n = len(qs)

    def table(counts, first):
        t = torch.zeros(len(counts), max(counts + [1]), dtype=torch.int32, device=dev)
        for i, c in enumerate(counts):
            t[i, :c] = ids[first:first + c]
            first += c
        return t

    counts = [x // ps for x in slots]
    s["table"] = table(counts[:n], 0)
    s["prefix_table"] = table(counts[n:], sum(counts[:n]))
    s["lens"] = torch.tensor([a + b for a, b in zip(qs, past)], dtype=torch.int32, device=dev)
    s["prefix_lens"] = torch.tensor(prefix, dtype=torch.int32, device=dev)
    starts = [0]
    for q in qs:
        starts.append(starts[-1] + q)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    groups = [0]
    for m in sizes:
        groups.append(groups[-1] + m)
    s["group_starts"] = torch.tensor(groups, dtype=torch.int32, device=dev)
    if case["op"] == "append":
        # rotation by the position in the cache
        s["positions"] = torch.cat([torch.arange(p, p + q, dtype=torch.int32, device=dev) for q, p in zip(qs, past)])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from lcm.nn import paged_attention as pa
        if "rot" in case:
            s["rope"] = pa.RotaryTable(s["cos"], s["sin"], style=case["style"])
            s["norm"] = None if case["norm"] == "none" else pa.HeadNorm(
                case["norm"], q_weight=s.get("qw"), k_weight=s.get("kw"), q_bias=s.get("qb"), k_bias=s.get("kb"), eps=_EPS)
        if case["op"] != "heads":
            qs, past, _, prefix = _shape(case)
            single = max(qs) == 1
            s["pages"] = pa.KVPages(s["k_pages"], s["v_pages"])
            s["batch"] = pa.PagedBatch(s["table"], s["lens"], None if single else s["starts"], max_q=max(qs),
                                       max_keys=max(a + b for a, b in zip(qs, past)))
            if case["op"] == "shared":
                s["prefix"] = pa.SharedPrefix(s["prefix_table"], s["prefix_lens"], s["group_starts"], max_keys=max(prefix))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------
def _norm(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "rms":
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    c = x - x.mean(-1, keepdim=True)
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    if w is not None:
        c = c * w.float()
    return c if b is None else c + b.float()


def _rotate(x, cos, sin, rot, style):
    """x: (rows, heads, d); cos, sin: (rows, rot / 2)."""
    cos, sin = cos[:, None, :], sin[:, None, :]
    part, rest = x[..., :rot], x[..., rot:]
    if style == "pairs":
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        part = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((part, rest), -1)


def _heads_plain(s, x, w, b):
    c = s["case"]
    pos = s["positions"].long()
    return _rotate(_norm(x.float(), c["norm"], w, b), s["cos"][pos], s["sin"][pos], c["rot"], c["style"]).to(x.dtype)


def _gather(pages, ids, length):
    """The first `length` positions of the pages `ids`: (heads, length, d) in 32 bits."""
    x = pages[ids.long()]
    return x.transpose(0, 1).flatten(1, 2)[:, :length].float()


def _attend_plain(q, k, v, past):
    """q: (rows, hq, d); k, v: (hk, keys, d); query j sees keys [0, past + j]."""
    rows, hq, d = q.shape
    hk, keys, _ = k.shape
    x = q.float().view(rows, hk, hq // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
    sc = torch.matmul(x, k.transpose(1, 2).contiguous()) * d ** -0.5
    if rows > 1:
        hidden = torch.arange(keys, device=q.device)[None, :] > past + torch.arange(rows, device=q.device)[:, None]
        sc = sc.view(hk, hq // hk, rows, keys).masked_fill(hidden, -math.inf).view(hk, -1, keys)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(hk, hq // hk, rows, d).permute(2, 0, 1, 3).reshape(rows, hq, d).to(q.dtype)


def _run_plain(s):
    c = s["case"]
    if c["op"] == "heads":
        return [_heads_plain(s, s["q"], s.get("qw"), s.get("qb")), _heads_plain(s, s["k"], s.get("kw"), s.get("kb"))]
    qs, past, sizes, prefix = _shape(c)
    ps = c["page"]
    if c["op"] == "append":
        q = _heads_plain(s, s["q"], s.get("qw"), s.get("qb"))
        k = _heads_plain(s, s["k"], s.get("kw"), s.get("kb"))
        seq = torch.searchsorted(s["starts"][1:].contiguous(), torch.arange(q.shape[0], device=q.device, dtype=torch.int32), right=True)
        at = s["lens"][seq].long() - (s["starts"][seq + 1] - torch.arange(q.shape[0], device=q.device)).long()
        page = s["table"][seq, at // ps].long()
        s["k_pages"][page, :, at % ps] = k
        s["v_pages"][page, :, at % ps] = s["v"]
        return [q, s["k_pages"], s["v_pages"]]
    outs, i, row = [], 0, 0
    for g, n in enumerate(sizes):
        if c["op"] == "shared":
            pk = _gather(s["k_pages"], s["prefix_table"][g, :-(-prefix[g] // ps)], prefix[g])
            pv = _gather(s["v_pages"], s["prefix_table"][g, :-(-prefix[g] // ps)], prefix[g])
        for b in range(i, i + n):
            length = qs[b] + past[b]
            ids = s["table"][b, :-(-length // ps)]
            k, v = _gather(s["k_pages"], ids, length), _gather(s["v_pages"], ids, length)
            if c["op"] == "shared":
                k, v = torch.cat((pk, k), 1), torch.cat((pv, v), 1)
            outs.append(_attend_plain(s["q"][row:row + qs[b]], k, v, past[b] + prefix[g]))
            row += qs[b]
        i += n
    return [torch.cat(outs)]


def run(state):
    if not own:
        return _run_plain(state)
    from lcm.nn import paged_attention as pa
    s = state
    op = s["case"]["op"]
    if op == "heads":
        return list(pa.head_norm_rope(s["q"], s["k"], positions=s["positions"], rope=s["rope"], norm=s["norm"]))
    if op == "append":
        q = pa.paged_append(s["pages"], s["batch"], s["k"], s["v"], q=s["q"], rope=s["rope"], norm=s["norm"])
        return [q, s["k_pages"], s["v_pages"]]
    if op == "attend":
        return [pa.paged_attention(s["q"], s["pages"], s["batch"])]
    return [pa.shared_prefix_attention(s["q"], s["pages"], s["batch"], s["prefix"])]


# ---- the same results from the definition, in 64 bits ----------------------------------------------------------------
def _exact_heads(s, x, w, b):
    """Norm, then every pair (x_i, x_j) of a head times exp(i angle) as one complex number."""
    c = s["case"]
    x = x.double()
    n, kind = x.shape[-1], c["norm"]
    if kind in ("standard", "unit"):
        x = x - x.sum(-1, keepdim=True) / n
    if kind != "none":
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / n + _EPS)
    if w is not None:
        x = x * w.double()
    if b is not None:
        x = x + b.double()
    half = c["rot"] // 2
    lanes = torch.arange(half, device=x.device)
    first, second = (2 * lanes, 2 * lanes + 1) if c["style"] == "pairs" else (lanes, lanes + half)
    pos = s["positions"].long()
    turn = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "heads":
        return [_exact_heads(s, s["q"], s.get("qw"), s.get("qb")), _exact_heads(s, s["k"], s.get("kw"), s.get("kb"))]
    qs, past, sizes, prefix = _shape(case)
    ps, hq, hk, d = case["page"], case["hq"], case["hk"], case["d"]
    if case["op"] == "append":
        k = _exact_heads(s, s["k"], s.get("kw"), s.get("kb"))
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        row = 0
        for b, (n, p) in enumerate(zip(qs, past)):
            at = torch.arange(p, p + n, device=k.device)
            page, off = s["table"][b].long()[at // ps], at % ps
            for pool, new in zip(pools, (k, s["v"].double())):
                pool[page, :, off] = new[row:row + n]
            row += n
        return [_exact_heads(s, s["q"], s.get("qw"), s.get("qb"))] + pools
    out = torch.empty(sum(qs), hq, d, dtype=torch.float64, device=s["q"].device)
    group = [g for g, n in enumerate(sizes) for _ in range(n)]
    row = 0
    for b, (n, p) in enumerate(zip(qs, past)):
        own_ids = s["table"][b, :-(-(n + p) // ps)].long()
        shared = prefix[group[b]]
        shared_ids = s["prefix_table"][group[b], :-(-shared // ps)].long()
        total = shared + n + p
        visible = shared + p + 1 + torch.arange(n, device=out.device)
        for h in range(hk):
            k, v = (torch.cat([x[shared_ids, h].reshape(-1, d)[:shared], x[own_ids, h].reshape(-1, d)[:n + p]]).double()
                    for x in (s["k_pages"], s["v_pages"]))
            for j in range(h * (hq // hk), (h + 1) * (hq // hk)):
                logits = (s["q"][row:row + n, j].double() @ k.T) / math.sqrt(d)
                if n > 1:
                    logits[torch.arange(total, device=out.device)[None] >= visible[:, None]] = -math.inf
                out[row:row + n, j] = torch.softmax(logits, -1) @ v
        row += n
    return [out]
