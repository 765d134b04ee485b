"""Plain 64-bit statements of the paged cache operators and the error bounds that their tests use.

Bounds count roundings: a rounding to a type is off by at most half a step, finfo(type).eps / 2 of the value; every fp32
operation by 2^-24 of its result."""

import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def heads(x, kind, w, b, eps, cos, sin, style, positions):
    """Norm and rotation of (rows, heads, d) in 64 bits; returns the result and a bound of the fp32 intermediates."""
    y = x.double()
    d = y.shape[-1]
    size = y.abs().amax(-1, keepdim=True)
    if kind in ("standard", "fp32", "unit"):
        y = y - y.mean(-1, keepdim=True)
    if kind is not None:
        r = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        y, size = y * r, size * r
    if w is not None:
        y, size = y * w.double(), size * w.double().abs().max()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs().max()
    if cos is not None:
        half = cos.shape[1]
        pos = positions.long().clamp(0, cos.shape[0] - 1)
        c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
        z = y.clone()
        if style == "pairs":
            e, o = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            z[..., 0:2 * half:2], z[..., 1:2 * half:2] = e * c - o * s, e * s + o * c
        else:
            e, o = y[..., :half], y[..., half:2 * half]
            z[..., :half], z[..., half:2 * half] = e * c - o * s, e * s + o * c
        y, size = z, 2 * size
    # norm: two sums over d values and a handful of operations; rotation: three more
    return y, (2 * d + 16) * U32 * size.expand_as(y)


def heads_bound(ref, slack, dtype):
    return half_step(dtype) * (ref.abs() + slack) + slack


def gather(pages, ids, count, page_size):
    """Positions [0, count) of a sequence (heads, count, d) in 64 bits and the mask of those whose page is there."""
    n = -(-count // page_size)
    ids = ids[:n].long()
    there = (ids >= 0) & (ids < pages.shape[0])
    x = pages[torch.where(there, ids, torch.zeros_like(ids))]
    x = x.transpose(0, 1).flatten(1, 2)[:, :count].double()
    return x, there.repeat_interleave(page_size)[:count]


def attend(q, k, v, there, visible, scale):
    """q (n, hq, d), k / v (hk, keys, d), there (keys,), visible (n,) keys of every row: the result in 64 bits and its bound in
    fp32 arithmetic with probabilities rounded to the operand type."""
    n, hq, d = q.shape
    hk, keys, _ = k.shape
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    mask = (torch.arange(keys, device=q.device)[None] < visible[:, None]) & there[None]
    for h in range(hq):
        kk, vv = k[h // (hq // hk)], v[h // (hq // hk)]
        for i in range(n):
            m = mask[i]
            if not bool(m.any()):
                continue
            x, kv, vals = q[i, h].double(), kk[m], vv[m]
            s = (kv @ x) * scale
            p = torch.softmax(s, 0)
            out[i, h] = p @ vals
            spread = p @ vals.abs()
            # a score: d products and sums, the scaling to base 2 and the subtraction of the maximum; exp2 itself 2 steps
            ds = (d + 8) * U32 * float((kv.abs() @ x.abs()).max()) * scale * 1.4427 + 4 * U32 * float(s.abs().max()) + 2 * U32
            many = (64 + math.ceil(int(m.sum()) / 16)) * U32
            bound[i, h] = spread * (2 * ds + half_step(q.dtype) + 2 * many)
    return out, bound


def attend_bound(ref, bound, dtype):
    return half_step(dtype) * (ref.abs() + bound) + bound


def paged(q, k_pages, v_pages, table, lens, starts, causal, scale, prefix=None):
    """The whole operator: (result, bound, rows that belong to a sequence).  prefix: (table, lens, group_starts)."""
    ps = k_pages.shape[2]
    rows = q.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    owned = torch.zeros(rows, dtype=torch.bool, device=q.device)
    starts = list(range(len(lens) + 1)) if starts is None else starts
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        if r1 <= r0:
            continue
        owned[r0:r1] = True
        length = min(length, table.shape[1] * ps)
        k, there = gather(k_pages, table[b], length, ps)
        v, _ = gather(v_pages, table[b], length, ps)
        visible = torch.arange(r0, r1, device=q.device) - r1 + length + 1 if causal else torch.full((r1 - r0,), length, device=q.device)
        visible = visible.clamp(min=0)
        if prefix is not None:
            for g in range(len(prefix[1])):
                if prefix[2][g] <= b < prefix[2][g + 1]:
                    n = prefix[1][g]
                    pk, pt = gather(k_pages, prefix[0][g], n, ps)
                    pv, _ = gather(v_pages, prefix[0][g], n, ps)
                    k, v, there, visible = torch.cat((pk, k), 1), torch.cat((pv, v), 1), torch.cat((pt, there)), visible + n
        out[r0:r1], bound[r0:r1] = attend(q[r0:r1], k, v, there, visible, scale)
    return out, bound, owned
