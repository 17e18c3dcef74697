"""A prompt's own attention and a drafted tree's restated on the CPU in float64 (imported by
their tests)."""

import torch

from oracle import attention as oatt
from oracle import codecs

PAGE, LATENT, PE, INDEX, HEADS = 64, 512, 64, 128, 64


def _bf16(v):
    return v.float().to(torch.bfloat16).double()


def index_query(x, pos, cos, sin):
    """(iq, iqs) of x [tokens, 64 * 128]."""
    i = torch.arange(INDEX)
    had = torch.tensor([[(-1.0) ** bin(int(a & b)).count("1") for b in i] for a in i], dtype=torch.float64)
    iq, iqs = torch.zeros(len(x), HEADS, INDEX // 2, dtype=torch.uint8), torch.zeros(len(x), HEADS, 4, dtype=torch.uint8)
    for n, p in enumerate(pos.tolist()):
        if not 0 <= p < len(cos):
            continue
        y = _bf16(x[n]).view(HEADS, INDEX)
        c, s = cos[p].double(), sin[p].double()
        a, b = y[:, :PE:2], y[:, 1:PE:2]
        y = torch.cat([_bf16(torch.stack([a * c - b * s, a * s + b * c], -1).flatten(1)), y[:, PE:]], -1)
        code, e8, _ = codecs.fp4_block_quant(_bf16(y @ had * INDEX**-0.5).float())
        iq[n], iqs[n] = codecs.e2m1_pack(code), e8
    return iq, iqs


def page_scores(iq, iqs, iw, req, pos, table, ikv, iks, columns):
    """(scores, the largest sum of a key's |weight x product|), f64 [tokens, columns]."""
    out = torch.full((len(iq), columns), -torch.inf, dtype=torch.float64)
    mag = torch.zeros(len(iq), columns, dtype=torch.float64)
    for n, (r, p) in enumerate(zip(req.tolist(), pos.tolist())):
        if not 0 <= r < len(table) or p < 0:
            continue
        q, w = oatt.index_query(iq[n], iqs[n]).double(), iw[n].double()
        for c in range(min(columns, table.shape[1], p // PAGE + 1)):
            if not 0 <= int(table[r, c]) < len(ikv):
                continue
            k = oatt.index_keys(ikv, iks, table[r, c:c + 1], min(PAGE, p + 1 - PAGE * c)).double()
            dot = q @ k.T
            terms = w[:, None] * torch.where(dot.isnan(), dot, dot.clamp_min(0))
            s = terms.sum(0)
            out[n, c] = torch.nan if bool(s.isnan().any()) else s.max()
            mag[n, c] = (w[:, None] * dot).abs().sum(0).max()
    return out, mag


def select_pages(scores, pos, picks, first, last):
    out = torch.full((len(scores), picks), -1, dtype=torch.int32)
    for n, p in enumerate(pos.tolist()):
        if p < 0:
            continue
        seen = min(p // PAGE + 1, scores.shape[1])
        bits = scores[n, :seen].contiguous().view(torch.int32).tolist()
        key = [b + 2**31 if b >= 0 else -1 - b for b in bits]
        forced = [c for c in range(seen) if c < first or c >= seen - last]
        rest = sorted((c for c in range(seen) if c not in forced), key=lambda c: (-key[c], c))
        ids = sorted(forced + rest[:picks - len(forced)])
        out[n, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return out


def _over(q, kv, kv_scale, slots, scale):
    """One token's attention over `slots` (any order, any number of times): (out, sum of p |v|,
    how far a logit may be off), f64. A logit: 578 roundings of f32 of its terms' magnitudes, and
    q's elements off by 2^-21.8 of their head's largest, in the last 64 dims by 2^-17.8."""
    rows = oatt.kv_rows(kv, kv_scale, slots).double()
    q = q.double()
    p = torch.softmax(q @ rows.T * scale, -1)
    k = rows.abs()
    off = 578 * 2.0**-24 * (q.abs() @ k.T) + q.abs().amax(-1, keepdim=True) * (2.0**-21.8 * k[:, :LATENT].sum(-1) + 2.0**-17.8 * k[:, LATENT:].sum(-1))
    return p @ rows[:, :LATENT], p @ k[:, :LATENT], float(off.max()) * abs(scale)


def _empty(q):
    return torch.zeros(*q.shape[:2], LATENT, dtype=torch.float64), torch.zeros(*q.shape[:2], LATENT, dtype=torch.float64), [0.0]


def attention(q, req, pos, pages, table, kv, kv_scale, scale):
    out, mag, top = _empty(q)
    for n, (r, p) in enumerate(zip(req.tolist(), pos.tolist())):
        if not 0 <= r < len(table):
            continue
        slots = []
        for c in pages[n].tolist():
            if 0 <= c < table.shape[1] and 0 <= int(table[r, c]) < len(kv) // PAGE:
                slots += [int(table[r, c]) * PAGE + j for j in range(PAGE) if c * PAGE + j <= p]
        if slots:
            out[n], mag[n], t = _over(q[n], kv, kv_scale, torch.tensor(slots), scale)
            top.append(t)
    return out, mag, max(top)


def tree_attention(q, starts, prefix, mask, table, kv, kv_scale, scale):
    out, mag, top = _empty(q)
    for r in range(len(prefix)):
        for n in range(int(starts[r]), int(starts[r + 1])):
            at = list(range(max(int(prefix[r]), 0))) + [max(int(prefix[r]), 0) + j for j in range(64) if int(mask[n]) >> j & 1]
            slots = [int(table[r, p // PAGE]) * PAGE + p % PAGE for p in at
                     if p // PAGE < table.shape[1] and 0 <= int(table[r, p // PAGE]) < len(kv) // PAGE]
            if slots:
                out[n], mag[n], t = _over(q[n], kv, kv_scale, torch.tensor(slots), scale)
                top.append(t)
    return out, mag, max(top)
