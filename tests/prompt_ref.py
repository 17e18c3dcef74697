"""The prompt-width operators restated on the CPU in float64 (imported by their tests)."""

import torch

from oracle import codecs

PAGE, LATENT, PE, INDEX = 64, 512, 64, 128


def rounded(x):
    """Rows as the values of their E4M3 codes and scales (one for each 128 columns), f64;
    a block that is not finite is NaN."""
    b = x.double().unflatten(-1, (-1, 128))
    a = b.abs().amax(-1, keepdim=True).clamp_min(2.0**-96)
    q = codecs.e4m3_decode((b * 448.0 / a).nan_to_num(0.0).clamp(-448, 448).float().to(torch.float8_e4m3fn)).double()
    return (torch.where(a.isfinite(), q * a / 448.0, torch.nan)).flatten(-2)


def weight(w, s):
    """A (16, 16)-laid E4M3 matrix [.., N, K] with its block scales as f64 values."""
    n, k = w.shape[-2:]
    v = codecs.e4m3_decode(codecs.aiter_unshuffle(w)).double()
    return v * s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def product(x, w, s):
    """(y, sum of |terms|) in f64."""
    xv, wv = rounded(x), weight(w, s)
    return xv @ wv.T, xv.abs() @ wv.abs().T


def experts(x, ids, wts, w13, s13, w2, s2, residual=None, shared=True):
    """(out, routed and shared sum, step) in f64; ``step`` [tokens] is what a token's output
    moves by, at most, when in each of its experts one mid's code moves by one: 32 / 448 of
    the largest mid (the widest step of E4M3 at its scale) times the largest weight."""
    xv, n = rounded(x), w13.shape[0] - bool(shared)
    y, step = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(len(x), dtype=torch.float64)

    def one(rows, e):
        g, u = (rows @ weight(w13[e], s13[e]).T).chunk(2, -1)
        mid, w = g * torch.sigmoid(g) * u, weight(w2[e], s2[e])
        return rounded(mid) @ w.T, mid.abs().amax(-1) * w.abs().max() * 32 / 448

    for e in sorted(set(ids.flatten().tolist()) & set(range(n))):
        t, j = (ids == e).nonzero(as_tuple=True)
        out, by = one(xv[t], e)
        y.index_add_(0, t, out * wts[t, j].double()[:, None])
        step.index_add_(0, t, by * wts[t, j].double().abs())
    if shared:
        out, by = one(xv, n)
        y, step = y + out, step + by
    return (y if residual is None else y + residual.double()), y, step


def _bf16(v):
    return v.float().to(torch.bfloat16).double()


def append(kv_a, ik, req, pos, table, caches, g_kv, g_ik, b_ik, cos, sin):
    """Apply the append to CPU copies of the caches (dict ikv, iks, kv, kv_scale) in place,
    token by token."""
    pages = caches["ikv"].shape[0]
    i = torch.arange(INDEX)
    had = torch.tensor([[(-1.0) ** bin(int(a & b)).count("1") for b in i] for a in i], dtype=torch.float64)
    for n in range(len(req)):
        r, p = int(req[n]), int(pos[n])
        if not (0 <= r < table.shape[0] and 0 <= p < min(len(cos), table.shape[1] * PAGE)):
            continue
        page, t = int(table[r, p // PAGE]), p % PAGE
        if not 0 <= page < pages:
            continue
        c, s = cos[p].double(), sin[p].double()

        def rot(v):
            a, b = v[0::2], v[1::2]
            return torch.stack([a * c - b * s, a * s + b * c], -1).flatten()

        x = kv_a[n].double()
        lat = x[:LATENT] / ((x[:LATENT] ** 2).mean() + 1e-6).sqrt() * g_kv.double()
        row = _bf16(torch.cat([lat, rot(x[LATENT:])]))
        slot = page * PAGE + t
        if caches["kv_scale"] is None:
            codes = row.clamp(-448, 448).float().to(torch.float8_e4m3fn)
        else:
            e = codecs.code_ceil((row.abs().amax().clamp_min(1e-4) / 448.0).float())
            scale = torch.exp2(e.double() - 127)
            caches["kv_scale"][slot] = scale.float()
            codes = (row / scale).float().to(torch.float8_e4m3fn)
        caches["kv"][slot] = codes.view(torch.uint8)

        k = ik[n].double()
        k = (k - k.mean()) / (k.var(correction=0) + 1e-6).sqrt() * g_ik.double() + b_ik.double()
        k = _bf16(torch.cat([rot(k[:PE]), k[PE:]]))
        k = _bf16(had @ k * INDEX**-0.5)
        code, e8, _ = codecs.fp4_block_quant(k.float())
        caches["ikv"][page, :, t] = codecs.e2m1_pack(code).reshape(4, 16)
        caches["iks"][page, :, t % 16 * 4 + t // 16] = e8
