"""A prompt's own attention over the paged caches, and a drafted tree's, operator by
operator, case by case.

* ``query``   index queries of a prompt's tokens: position rotation, Hadamard and FP4
* ``scores``  the cheap score of every page of a token's request: the largest of its keys'
  index scores
* ``select``  the pages that a token's query reads: its own and the best-scored, lowest first
* ``attend``  sparse MLA attention of a token over the keys of its selected pages
* ``tree``    MLA attention of a tree of drafted tokens over its request's keys and, of the
  draft, those that each token's mask lets it see

Pages hold 64 keys: an E4M3 row of 512 latent and 64 rotated dims with an f32 scale (or raw),
and an FP4 index key of 128 dims with a scale for each 32, as the decode launches read them.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE, LATENT, PE, INDEX, INDEX_HEADS = 64, 512, 64, 128, 64
ROW = LATENT + PE
SCALE = 192**-0.5  # (128 + 64)^-1/2: the width of a query before it is absorbed
E4M3 = torch.float8_e4m3fn
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's index query: only latency counts
        dict(name="query_1", op="query", tokens=1, start=20000, f32=False, wide=0),
        # a full prefill chunk's, a slice of a wider projection
        dict(name="query_8192", op="query", tokens=8192, start=0, f32=False, wide=128),
        # a chain of drafted tokens behind a long request
        dict(name="scores_9", op="scores", tokens=9, requests=1, start=20000, pads=0),
        # a full prefill chunk from a prompt's first token on
        dict(name="scores_8192", op="scores", tokens=8192, requests=1, start=0, pads=0),
        # the chain's pages
        dict(name="select_9", op="select", tokens=9, columns=313, start=20000, picks=32, first=0, last=1),
        # a full chunk's, late in a prompt of 32768 tokens
        dict(name="select_8192", op="select", tokens=8192, columns=512, start=24576, picks=32, first=1, last=2),
        # one token behind a long request
        dict(name="attend_1", op="attend", tokens=1, requests=1, start=20000, pads=0, heads=32, picks=32, raw=False),
        # a batch of ragged prompts over raw rows, half as many heads a GPU
        dict(name="attend_777", op="attend", tokens=777, requests=5, start=900, pads=7, heads=16, picks=32, raw=True),
        # a prefill chunk behind 8192 tokens
        dict(name="attend_4096", op="attend", tokens=4096, requests=1, start=8192, pads=0, heads=32, picks=32, raw=False),
        # a small tree behind a long request
        dict(name="tree_5", op="tree", requests=1, nodes=5, prefix=20000, heads=32, raw=False, even=False),
        # a few requests' trees of unequal sizes behind unequal prefixes
        dict(name="tree_7x33", op="tree", requests=7, nodes=33, prefix=3001, heads=32, raw=True, even=False),
        # a decoding batch, each request with a tree of 32
        dict(name="tree_32x32", op="tree", requests=32, nodes=32, prefix=8000, heads=32, raw=False, even=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["query", "scores", "select", "attend", "tree"])
    if op == "query":
        f32 = rng.random() < 0.4
        return dict(op=op, tokens=log(1, 4000 if f32 else 8000), start=log(1, 30000) if rng.random() < 0.5 else 0, f32=f32,
                    wide=8 * rng.randint(1, 99) if rng.random() < 0.4 else 0)
    if op == "scores":
        tokens = log(1, 8000)
        return dict(op=op, tokens=tokens, requests=min(tokens, log(1, 16)), start=log(1, min(30000, 30_000_000 // tokens)) // 2,
                    pads=rng.choice([0, 0, rng.randint(1, 40)]))
    if op == "select":
        tokens = log(1, 8000)
        columns = log(1, min(2000, 4_000_000 // tokens))
        first, last = rng.randint(0, 2), rng.randint(0, 2)
        return dict(op=op, tokens=tokens, columns=columns, start=rng.randint(0, PAGE * columns), picks=first + last + log(1, 64),
                    first=first, last=last)
    if op == "attend":
        heads, picks = rng.choice([8, 16, 32, 32, 32, 64, 128]), log(1, 64)
        tokens = log(1, min(6000, 120_000 // picks * 32 // max(heads, 32)))
        return dict(op=op, tokens=tokens, requests=min(tokens, log(1, 16)), start=log(1, 16000) if rng.random() < 0.7 else 0,
                    pads=rng.choice([0, 0, rng.randint(1, 9)]), heads=heads, picks=picks, raw=rng.random() < 0.4)
    heads, requests, nodes = rng.choice([8, 16, 32, 32, 32, 64, 128]), log(1, 32), log(1, 64)
    return dict(op=op, requests=requests, nodes=nodes, prefix=log(1, min(30000, 7_500_000 // (nodes * requests) * 32 // max(heads, 32))),
                heads=heads, raw=rng.random() < 0.4, even=rng.random() < 0.5)


# --------------------------------------------------------------------- inputs


def _spans(case):
    """Each request's first position and length: unequal shares of the call's tokens."""
    t, r = case["tokens"] - min(case["pads"], case["tokens"] - 1), min(case["requests"], case["tokens"])
    cuts = [round(t * (j / r) ** 1.5) for j in range(r + 1)]
    return [(case["start"] * (j + 1) // r, cuts[j + 1] - cuts[j]) for j in range(r)]


def _trees(case):
    """Each request's prefix and number of drafted tokens."""
    r = case["requests"]
    if case["even"]:
        return [(case["prefix"], case["nodes"])] * r
    return [(case["prefix"] * (j + 1) // r, max(1, case["nodes"] * (r - j) // r)) for j in range(r)]


def _table(used, g, dev):
    """Page tables of requests of `used` pages each, in no order; page 0 is nobody's."""
    order = torch.randperm(sum(used) + 1, generator=g, device=dev).to(torch.int32) + 1
    table = torch.zeros(len(used), max(used), dtype=torch.int32, device=dev)
    at = 0
    for j, u in enumerate(used):
        table[j, :u] = order[at:at + u]
        at += u
    return table, sum(used) + 2


def _grid(lengths, dev):
    """[requests, longest] places of each request's rows among the packed ones; -1: none."""
    grid = torch.full((len(lengths), max(lengths)), -1, dtype=torch.long)
    at = 0
    for j, n in enumerate(lengths):
        grid[j, :n] = torch.arange(at, at + n)
        at += n
    return grid.to(dev)


def _tokens(case, g, dev):
    """Request and position of each token (pads: -1), the requests' page tables, the pool's
    pages and the tokens by request."""
    spans, t = _spans(case), case["tokens"]
    req = torch.full((t,), -1, dtype=torch.int32)
    pos = torch.full((t,), -1, dtype=torch.int32)
    at = 0
    for j, (first, n) in enumerate(spans):
        req[at:at + n] = j
        pos[at:at + n] = torch.arange(first, first + n, dtype=torch.int32)
        at += n
    table, pages = _table([-(-(first + n) // PAGE) or 1 for first, n in spans], g, dev)
    return req.to(dev), pos.to(dev), table, pages, _grid([n for _, n in spans], dev)


def _rope(n, dev):
    angle = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
        -torch.arange(0, PE, 2, dtype=torch.float64, device=dev) / PE)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _latent_pool(pages, raw, g, dev):
    kv = torch.randn(pages * PAGE, ROW, generator=g, device=dev).to(E4M3).view(torch.uint8)
    return kv, None if raw else 2.0 ** torch.randint(-2, 2, (pages * PAGE,), generator=g, device=dev).float()


def _picked(pos, columns, picks, g, dev):
    """The page lists of tokens at `pos`, ascending: the token's own page and others by a score
    that drifts slowly from token to token, as those of a text do."""
    t = len(pos)
    base = torch.randn(-(-t // 64) + 1, columns, generator=g, device=dev).repeat_interleave(64, 0)[:t]
    score = base + 0.4 * torch.randn(t, columns, generator=g, device=dev)
    page, last = torch.arange(columns, device=dev), pos[:, None] // PAGE
    score = torch.where(page < last, score, torch.where(page == last, torch.inf, -torch.inf))
    k = min(picks, columns)
    top = score.topk(k, -1)
    ids = torch.where(top.values > -torch.inf, top.indices, 1 << 30).sort(-1).values
    ids = torch.where(ids < 1 << 30, ids, -1).to(torch.int32)
    return torch.cat([ids, torch.full((t, picks - k), -1, dtype=torch.int32, device=dev)], 1) if k < picks else ids.contiguous()


def _masks(trees, rng, dev):
    """Each drafted token's ancestors and itself as bits, of trees whose tokens hang from one
    of the few before them."""
    out = []
    for _, n in trees:
        seen = []
        for i in range(n):
            up = int(rng[len(out) % len(rng)] * 4) + 1
            seen.append((seen[i - up] if i >= up else 0) | 1 << i)
            out.append(seen[i] - (1 << 64 if seen[i] >= 1 << 63 else 0))
    return torch.tensor(out, dtype=torch.int64).to(dev)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if op == "query":
        t, dtype = case["tokens"], torch.float32 if case["f32"] else torch.bfloat16
        cos, sin = _rope(case["start"] + t, dev)
        return dict(op=op, x=(1.5 * randn(t, case["wide"] + INDEX_HEADS * INDEX)).to(dtype)[:, case["wide"]:], cos=cos, sin=sin,
                    pos=torch.arange(case["start"], case["start"] + t, dtype=torch.int32, device=dev))
    if op == "select":
        t, n = case["tokens"], case["columns"]
        pos = (case["start"] + torch.arange(t, device=dev)).clamp_max(n * PAGE - 1).to(torch.int32)
        scores = torch.where(torch.arange(n, device=dev) <= pos[:, None] // PAGE, 0.3 * randn(t, n) + 0.2, -torch.inf)
        return dict(op=op, scores=scores, pos=pos, picks=case["picks"], first=case["first"], last=case["last"])
    if op == "tree":
        trees = _trees(case)
        lengths = [n for _, n in trees]
        table, pages = _table([-(-(p + n) // PAGE) for p, n in trees], g, dev)
        kv, kv_scale = _latent_pool(pages, case["raw"], g, dev)
        starts = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32)
        return dict(op=op, q=randn(sum(lengths), case["heads"], ROW).to(torch.bfloat16), starts=starts.to(dev),
                    prefix=torch.tensor([p for p, _ in trees], dtype=torch.int32).to(dev),
                    mask=_masks(trees, torch.rand(257, generator=g, device=dev).tolist(), dev), table=table, kv=kv,
                    kv_scale=kv_scale, grid=_grid(lengths, dev))
    req, pos, table, pages, grid = _tokens(case, g, dev)
    t = case["tokens"]
    if op == "scores":
        return dict(op=op, iq=torch.randint(0, 256, (t, INDEX_HEADS, INDEX // 2), generator=g, device=dev, dtype=torch.uint8),
                    iqs=torch.randint(125, 129, (t, INDEX_HEADS, 4), generator=g, device=dev, dtype=torch.uint8),
                    iw=(0.01 * randn(t, INDEX_HEADS)).to(torch.bfloat16), req=req, pos=pos, table=table, grid=grid,
                    ikv=torch.randint(0, 256, (pages, 4, PAGE, 16), generator=g, device=dev, dtype=torch.uint8),
                    iks=torch.randint(124, 130, (pages, 4, PAGE), generator=g, device=dev, dtype=torch.uint8))
    kv, kv_scale = _latent_pool(pages, case["raw"], g, dev)
    return dict(op=op, q=randn(t, case["heads"], ROW).to(torch.bfloat16), req=req, pos=pos, table=table, kv=kv, kv_scale=kv_scale,
                pages=_picked(pos, table.shape[1], case["picks"], g, dev))


# ----------------------------------------------------------------- the passes


def run(s):
    return {"query": _query, "scores": _scores, "select": _select, "attend": _attend, "tree": _tree}[s["op"]](s)


def _query(s):
    if own:
        from sgl_amd_mono_amd import prompt

        return prompt.index_query(s["x"], s["pos"], s["cos"], s["sin"])
    # in f64 up to each rounding: a four-bit code is a border's width from another
    pos, t = s["pos"].long(), len(s["pos"])
    x = s["x"].to(torch.bfloat16).double().view(t, INDEX_HEADS, INDEX)
    cos, sin = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
    a, b = x[..., 0:PE:2], x[..., 1:PE:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    x = torch.cat([turned.float().to(torch.bfloat16).double(), x[..., PE:]], -1)
    i = torch.arange(INDEX, device=x.device)
    bits = ((i[:, None] & i)[..., None] >> torch.arange(7, device=x.device) & 1).sum(-1)
    x = (x @ (1.0 - 2.0 * (bits % 2)).double() * INDEX**-0.5).float().to(torch.bfloat16).float().unflatten(-1, (4, 32))
    need, up = torch.frexp(x.abs().amax(-1).clamp_min(6.0 * 2.0**-126) / 6.0)
    e8 = (up + 127 - (need == 0.5).int()).clamp(1, 254)
    v = x / torch.ldexp(torch.ones_like(need), e8 - 127)[..., None]
    m = v.abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    code = code + 8 * ((v < 0) & (code > 0))
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8).flatten(-2), e8.to(torch.uint8)


def _fp4(packed, scales):
    """Values of E2M1 pairs [.., n / 2] with an E8M0 scale for each 32."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    size = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return level[code] * size.repeat_interleave(32, -1)


def _index_keys(s):
    """Every request's index keys by position, f32 [requests, keys, 128]."""
    page = s["table"].long()
    packed = s["ikv"][page].transpose(2, 3).flatten(-2)  # [requests, pages, 64, 64]
    t = torch.arange(PAGE, device=page.device)
    return _fp4(packed, s["iks"][page][..., t % 16 * 4 + t // 16].transpose(2, 3)).flatten(1, 2)


def _scores(s):
    if own:
        from sgl_amd_mono_amd import attn, prompt

        caches = attn.AttnCaches(ikv=s["ikv"], iks=s["iks"], kv=None, kv_scale=None)
        return prompt.page_scores(s["iq"], s["iqs"], s["iw"], s["req"], s["pos"], s["table"], caches)
    (r, n), t, columns = s["grid"].shape, len(s["pos"]), s["table"].shape[1]
    at = s["grid"].clamp_min(0)
    q = _fp4(s["iq"], s["iqs"])[at].flatten(1, 2)  # [requests, tokens x heads, 128]
    dot = torch.bmm(q, _index_keys(s).transpose(1, 2).contiguous()).view(r, n, INDEX_HEADS, -1)
    score = dot.relu_().mul_(s["iw"].float()[at][..., None]).sum(2)  # [requests, tokens, keys]
    live = torch.arange(columns * PAGE, device=at.device) <= s["pos"][at][..., None]
    best = torch.where(live, score, -torch.inf).unflatten(-1, (columns, PAGE)).amax(-1)
    out = torch.full((t + 1, columns), -torch.inf, device=at.device)
    out[torch.where(s["grid"] >= 0, s["grid"], t)] = best
    return out[:t]


def _select(s):
    if own:
        from sgl_amd_mono_amd import prompt

        return prompt.select_pages(s["scores"], s["pos"], s["picks"], first=s["first"], last=s["last"])
    t, n = s["scores"].shape
    page, own_page = torch.arange(n, device=s["pos"].device), (s["pos"][:, None] // PAGE).clamp_max(n - 1)
    # whole numbers in the scores' order, those always taken above every score
    b = s["scores"].view(torch.int32).long()
    key = torch.where(b >= 0, b + (1 << 31), -1 - b & 0xFFFFFFFF)
    always = (page < s["first"]) | (page > own_page - s["last"])
    key = torch.where(page <= own_page, torch.where(always, 1 << 33, key), -1)
    order = key.sort(stable=True, dim=-1, descending=True)
    k = min(n, s["picks"])
    ids = torch.where(order.values[:, :k] >= 0, order.indices[:, :k], n).sort(-1).values
    ids = torch.where(ids < n, ids, -1).to(torch.int32)
    return torch.cat([ids, torch.full((t, s["picks"] - k), -1, dtype=torch.int32, device=ids.device)], 1)


def _rows(s, slot):
    rows = s["kv"].view(E4M3)[slot].float()
    return rows if s["kv_scale"] is None else rows.mul_(s["kv_scale"][slot][..., None])


def _softmax(logits, seen):
    logits = torch.where(seen, logits, -torch.inf)
    e = (logits - logits.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
    return e / e.sum(-1, keepdim=True).clamp_min(1e-38)  # a row that sees nothing: zeros


def _attend(s):
    if own:
        from sgl_amd_mono_amd import attn, prompt

        caches = attn.AttnCaches(ikv=None, iks=None, kv=s["kv"], kv_scale=s["kv_scale"])
        return prompt.attention(s["q"], s["req"], s["pos"], s["pages"], s["table"], caches, softmax_scale=SCALE)
    key = (s["pages"].long()[..., None] * PAGE + torch.arange(PAGE, device=s["q"].device)).flatten(1)  # [tokens, picks x 64]
    seen = (key >= 0) & (key <= s["pos"][:, None]) & (s["req"][:, None] >= 0)
    page = s["table"].long()[s["req"].long().clamp_min(0)[:, None], torch.where(seen, key // PAGE, 0)]
    rows = _rows(s, page * PAGE + key % PAGE)
    p = _softmax(torch.bmm(s["q"].float(), rows.transpose(1, 2)) * SCALE, seen[:, None])
    return torch.bmm(p, rows[..., :LATENT]).to(torch.bfloat16)


def _tree(s):
    if own:
        from sgl_amd_mono_amd import attn, prompt

        caches = attn.AttnCaches(ikv=None, iks=None, kv=s["kv"], kv_scale=s["kv_scale"])
        return prompt.tree_attention(s["q"], s["starts"], s["prefix"], s["mask"], s["table"], caches, softmax_scale=SCALE)
    (r, n), heads, nodes = s["grid"].shape, s["q"].shape[1], len(s["q"])
    at = s["grid"].clamp_min(0)
    key = torch.arange(s["table"].shape[1] * PAGE, device=at.device)
    rows = _rows(s, s["table"].long()[:, key // PAGE] * PAGE + key % PAGE)  # [requests, keys, 576]
    behind = key - s["prefix"][:, None]  # [requests, keys]: the place among the drafted
    bit = s["mask"][at][..., None] >> behind.clamp(0, 63)[:, None] & 1
    seen = (behind < 0)[:, None] | ((behind < 64)[:, None] & (bit != 0))  # [requests, nodes, keys]
    logits = torch.bmm(s["q"].float()[at].flatten(1, 2), rows.transpose(1, 2)) * SCALE
    p = _softmax(logits.view(r, n, heads, -1), seen[:, :, None])
    o = torch.bmm(p.flatten(1, 2), rows[..., :LATENT]).view(r, n, heads, LATENT)
    out = torch.empty(nodes + 1, heads, LATENT, dtype=torch.bfloat16, device=at.device)
    out[torch.where(s["grid"] >= 0, s["grid"], nodes)] = o.to(torch.bfloat16)
    return out[:nodes]


def work(case):
    op = case["op"]
    if op == "query":
        t = case["tokens"]
        per = INDEX_HEADS * (INDEX * (4 if case["f32"] else 2) + INDEX // 2 + 4) + 4 + 4 * PE
        return dict(bytes=t * per, flops=t * INDEX_HEADS * INDEX * 12)
    if op == "select":
        live = sum(min(case["columns"], (case["start"] + i) // PAGE + 1) for i in range(case["tokens"]))
        return dict(bytes=4 * live + 4 * case["tokens"] * (case["picks"] + 1), flops=live)
    if op == "tree":
        trees = _trees(case)
        row, h = ROW + (0 if case["raw"] else 4), case["heads"]
        # a tree hangs from one of the four before: a token sees some fifth of its request's others
        keys = sum(n * (p + max(1, n // 5)) for p, n in trees)
        return dict(bytes=sum((p + n) * row + n * (2 * h * (ROW + LATENT) + 8) for p, n in trees), flops=2 * h * (ROW + LATENT) * keys)
    spans, t = _spans(case), case["tokens"]
    if op == "scores":
        keys, pairs = sum(a + n for a, n in spans), sum(n * a + n * (n + 1) // 2 for a, n in spans)
        columns = max(-(-(a + n) // PAGE) for a, n in spans)
        per = INDEX_HEADS * (INDEX // 2 + 4 + 2) + 8 + 4 * columns
        return dict(bytes=keys * (INDEX // 2 + 4) + t * per, flops=2 * INDEX_HEADS * INDEX * pairs)
    h, most, pairs = case["heads"], case["picks"] * PAGE, 0
    for a, n in spans:
        for i in range(a, a + n):
            pairs += i + 1 if i // PAGE < case["picks"] else most - PAGE + i % PAGE + 1
    keys = min(pairs, sum(a + n for a, n in spans))
    row = ROW + (0 if case["raw"] else 4)
    return dict(bytes=keys * row + t * (2 * h * (ROW + LATENT) + 8 + 4 * case["picks"]), flops=2 * h * (ROW + LATENT) * pairs)


# ------------------------------------------------------- the results in 64 bits


def _bf16_of(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-120))) - 7.0)
    return torch.round(v / step) * step


def _fp4_of(packed, scales):
    """One row of E2M1 pairs each and its E8M0 scales as f64 values, by their exponents."""
    code = torch.empty(*packed.shape[:-1], 2 * packed.shape[-1], dtype=torch.long, device=packed.device)
    code[..., 0::2], code[..., 1::2] = packed % 16, packed // 16
    e, m = code % 8 // 2, code % 2
    v = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2(e.double() - 1.0))
    v = torch.where(code >= 8, -v, v).unflatten(-1, (-1, 32))
    return (v * torch.exp2(scales.double() - 127.0)[..., None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    return {"query": _exact_query, "scores": _exact_scores, "select": _exact_select, "attend": _exact_attend,
            "tree": _exact_tree}[case["op"]](s)


def _exact_query(s):
    t = len(s["pos"])
    x = _bf16_of(s["x"].double()).view(t, INDEX_HEADS, INDEX)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]
    pairs = torch.view_as_complex(x[..., :PE].unflatten(-1, (-1, 2)).contiguous())
    y = torch.cat([_bf16_of(torch.view_as_real(pairs * turn).flatten(-2)), x[..., PE:]], -1)
    for h in (1, 2, 4, 8, 16, 32, 64):
        y = y.reshape(t, INDEX_HEADS, INDEX // (2 * h), 2, h)
        y = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], 3)
    y = _bf16_of(y.reshape(t, INDEX_HEADS, 4, 32) / INDEX**0.5)
    e8 = torch.ceil(torch.log2(y.abs().amax(-1) / 6.0)).clamp(-126.0, 127.0)
    v = (y / torch.exp2(e8)[..., None]).abs()
    # below 2 the values are halves, below 4 whole, below 6 even: rounded to even multiples of the step
    step = torch.where(v < 2.0, 0.5, torch.where(v < 4.0, 1.0, 2.0))
    near = torch.round(v / step) * step
    level = torch.tensor(LEVELS, dtype=torch.float64, device=v.device)
    code = torch.searchsorted(level, near)
    code = code + 8 * ((y < 0) & (code > 0))
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8).flatten(-2), (e8 + 127).to(torch.uint8)


def _exact_scores(s):
    out = torch.full((len(s["pos"]), s["table"].shape[1]), -torch.inf, dtype=torch.float64, device=s["pos"].device)
    k = torch.arange(PAGE, device=out.device)
    for r in range(len(s["table"])):
        mine = (s["req"] == r).nonzero().flatten()
        page = s["table"][r].long()
        keys = torch.stack([_fp4_of(s["ikv"][page][:, c], s["iks"][page][:, c, k % 16 * 4 + k // 16][..., None]) for c in range(4)], 2)
        keys = keys.reshape(-1, INDEX)
        for at in mine.split(256):
            q = _fp4_of(s["iq"][at], s["iqs"][at])
            score = torch.zeros(len(at), len(keys), dtype=torch.float64, device=out.device)
            for h in range(INDEX_HEADS):
                score += (q[:, h] @ keys.T).clamp_min(0) * s["iw"][at, h].double()[:, None]
            score.masked_fill_(torch.arange(len(keys), device=out.device) > s["pos"][at, None], -torch.inf)
            out[at] = score.view(len(at), -1, PAGE).amax(-1)
    return out


def _exact_select(s):
    scores, pos, t = s["scores"].cpu().double(), s["pos"].cpu().long(), len(s["pos"])
    n = scores.shape[1]
    mine = (pos // PAGE).clamp_max(n - 1)
    page = torch.arange(n).expand(t, n)
    taken = (page < s["first"]) | (page > mine[:, None] - s["last"])
    value = torch.where(taken, torch.inf, scores.clamp(-1e300, 1e300)).masked_fill(page > mine[:, None], -torch.inf)
    order = value.argsort(dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(1, order, page.contiguous())
    keep = (rank < s["picks"]) & (page <= mine[:, None])
    out = torch.full((t, s["picks"]), -1, dtype=torch.int32)
    row, col = keep.nonzero(as_tuple=True)
    out[row, (keep.cumsum(-1) - 1)[row, col]] = col.to(torch.int32)
    return out.to(s["pos"].device)


def _exact_rows(s, slot):
    return s["kv"][slot].view(E4M3).double() * (1.0 if s["kv_scale"] is None else s["kv_scale"][slot].double()[..., None])


def _exact_attend(s):
    (t, h), pages, pos = s["q"].shape[:2], s["pages"].long(), s["pos"].long()
    out = torch.zeros(t, h, LATENT, dtype=torch.float64, device=pos.device)
    k = torch.arange(PAGE, device=pos.device)
    for at in (s["req"] >= 0).nonzero().flatten().split(128):
        page = pages[at].clamp_min(0)
        seen = ((pages[at] >= 0)[..., None] & (page[..., None] * PAGE + k <= pos[at, None, None])).flatten(1)
        slot = (s["table"].long()[s["req"][at].long()[:, None], page.clamp_max(s["table"].shape[1] - 1)][..., None] * PAGE + k).flatten(1)
        rows = _exact_rows(s, slot)
        logits = torch.matmul(s["q"][at].double(), rows.transpose(1, 2).contiguous()) * SCALE
        p = torch.softmax(logits.masked_fill(~seen[:, None], -torch.inf), -1)
        out[at] = torch.matmul(p, rows[..., :LATENT].contiguous())
    return out


def _exact_tree(s):
    q, mask = s["q"].double(), s["mask"].tolist()
    starts, prefix = s["starts"].tolist(), s["prefix"].tolist()
    out = torch.zeros(*q.shape[:2], LATENT, dtype=torch.float64, device=q.device)
    for r, p in enumerate(prefix):
        a, b = starts[r], starts[r + 1]
        key = torch.arange(p + b - a, device=q.device)
        rows = _exact_rows(s, s["table"][r].long()[key // PAGE] * PAGE + key % PAGE)
        seen = torch.ones(b - a, len(key), dtype=torch.bool)
        seen[:, p:] = torch.tensor([[mask[i] >> j & 1 for j in range(b - a)] for i in range(a, b)], dtype=torch.bool)
        logits = (q[a:b] @ rows.T * SCALE).masked_fill(~seen.to(q.device)[:, None], -torch.inf)
        out[a:b] = torch.softmax(logits, -1) @ rows[:, :LATENT]
    return out
