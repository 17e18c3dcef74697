"""The refusals of a prompt's own attention and a drafted tree's: argument checks run before
any GPU call, so they are testable on the CPU (pointers that no check lets through are never
used)."""

import ctypes as C

import pytest
import torch

import pages_ref as ref
from oracle import attention as oatt
from oracle import layer as olayer
from sgl_amd_mono_amd import _lib, prompt
from sgl_amd_mono_amd.attn import AttnCaches

P = 1 << 20  # an aligned address that is nobody's


def _call(fn, cls, a, kw):
    a = {**a, **kw}
    return _lib.check(getattr(_lib.lib(), fn)(C.byref(cls(**a)), None))


QUERY = dict(x=P, x_stride=8192, f32=0, tokens=3, pos=P, max_pos=9, rope_cos=P, rope_sin=P, iq=P, iqs=P)


@pytest.mark.parametrize("kw,what", [
    (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 20) + 1), "tokens"), (dict(max_pos=-1), "max_pos"), (dict(max_pos=0), "max_pos"),
    (dict(x_stride=8191), "x_stride"), (dict(x_stride=8196), "x_stride"), (dict(x_stride=8194, f32=1), "x_stride"),
    (dict(x=None), "x must"), (dict(x=P + 8), "x must"), (dict(pos=None), "pos"), (dict(rope_cos=None), "rope_cos"),
    (dict(rope_sin=P + 4), "rope_sin"), (dict(iq=None), "iq must"), (dict(iqs=None), "iqs"),
])  # fmt: skip
def test_query_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _call("mono_prompt_query", _lib.PromptQueryArgs, QUERY, kw)


SCORES = dict(iq=P, iqs=P, iw=P, tokens=3, req=P, pos=P, page_table=P, requests=2, pt_stride=4, n_pages=8, ikv=P, iks=P, out=P, columns=4)


@pytest.mark.parametrize("kw,what", [
    (dict(tokens=-1), "tokens"), (dict(requests=-1), "requests"), (dict(pt_stride=-1), "pt_stride"), (dict(n_pages=-1), "n_pages"),
    (dict(columns=-1), "columns"), (dict(columns=8193), "columns"), (dict(iq=P + 8), "iq must"), (dict(iqs=None), "iqs"),
    (dict(iw=P + 4), "iw"), (dict(req=None), "req"), (dict(pos=None), "pos"), (dict(page_table=None), "page_table"),
    (dict(ikv=None), "ikv"), (dict(iks=P + 2), "iks"), (dict(out=None), "out"),
])  # fmt: skip
def test_scores_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _call("mono_prompt_scores", _lib.PromptScoresArgs, SCORES, kw)


SELECT = dict(scores=P, stride=9, tokens=3, columns=9, pos=P, picks=4, first=1, last=1, pages=P)


@pytest.mark.parametrize("kw,what", [
    (dict(tokens=-1), "tokens"), (dict(columns=0), "columns"), (dict(columns=8193), "columns"), (dict(picks=0), "picks"),
    (dict(picks=8193), "picks"), (dict(first=-1), "first and last"), (dict(last=-1), "first and last"),
    (dict(first=3, last=2), "first and last"), (dict(first=(1 << 31) - 1, last=(1 << 31) - 1), "first and last"),
    (dict(stride=8), "stride"), (dict(scores=None), "scores"), (dict(pos=None), "pos"), (dict(pages=None), "pages"),
])  # fmt: skip
def test_select_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _call("mono_prompt_select", _lib.PromptSelectArgs, SELECT, kw)


POOL = dict(page_table=P, requests=2, pt_stride=40, n_pages=8, kv=P, kv_scale=P, softmax_scale=0.1, out=P, workspace=P, workspace_bytes=1 << 30)
ATTEND = dict(q=P, tokens=3, heads=32, req=P, pos=P, pages=P, picks=32, **POOL)
TREE = dict(q=P, nodes=3, heads=32, starts=P, prefix=P, mask=P, **POOL)
SHARED = [
    (dict(heads=0), "heads"), (dict(heads=129), "heads"), (dict(requests=-1), "requests"), (dict(pt_stride=-1), "pt_stride"),
    (dict(n_pages=-1), "n_pages"), (dict(q=None), "q must"), (dict(q=P + 8), "q must"), (dict(page_table=None), "page_table"),
    (dict(kv=P + 8), "kv must"), (dict(kv_scale=P + 4), "kv_scale"), (dict(out=None), "out"), (dict(out=P + 8), "out"),
    (dict(softmax_scale=float("nan")), "softmax_scale"), (dict(softmax_scale=float("inf")), "softmax_scale"),
    (dict(softmax_scale=3e38), "softmax_scale"),
    (dict(workspace=None), "workspace"), (dict(workspace=P + 16), "workspace"), (dict(workspace_bytes=100), "workspace must hold"),
]  # fmt: skip


@pytest.mark.parametrize("kw,what", SHARED + [
    (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 20) + 1), "tokens"), (dict(picks=-1), "picks"), (dict(picks=8193), "picks"),
    (dict(req=None), "req"), (dict(pos=None), "pos"), (dict(pages=None), "pages"),
])  # fmt: skip
def test_attention_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _call("mono_prompt_attention", _lib.PromptAttentionArgs, ATTEND, kw)


@pytest.mark.parametrize("kw,what", SHARED + [
    (dict(nodes=-1), "nodes"), (dict(nodes=(1 << 20) + 1), "nodes"), (dict(starts=None), "starts"), (dict(prefix=None), "prefix"),
    (dict(mask=P + 4), "mask"),
])  # fmt: skip
def test_tree_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _call("mono_prompt_tree", _lib.PromptTreeArgs, TREE, kw)


def test_calls_of_no_rows_look_at_nothing():
    for fn, cls, a, rows in (("query", _lib.PromptQueryArgs, QUERY, "tokens"), ("scores", _lib.PromptScoresArgs, SCORES, "tokens"),
                             ("select", _lib.PromptSelectArgs, SELECT, "tokens"), ("attention", _lib.PromptAttentionArgs, ATTEND, "tokens"),
                             ("tree", _lib.PromptTreeArgs, TREE, "nodes")):  # fmt: skip
        none = {k: None if v == P else v for k, v in a.items()}
        _call(f"mono_prompt_{fn}", cls, none, {rows: 0})


def test_null_args():
    h = _lib.lib()
    for fn in (h.mono_prompt_query, h.mono_prompt_scores, h.mono_prompt_select, h.mono_prompt_attention, h.mono_prompt_tree):
        with pytest.raises(ValueError, match="args is NULL"):
            _lib.check(fn(None, None))


def test_append_at_refuses_a_bad_pointer():
    a = dict(kv_a=P, kv_stride=576, ik=P, ik_stride=128, f32=0, tokens=3, req=P, pos=P, page_table=P, requests=2, pt_stride=4,
             n_pages=8, max_pos=100, g_kv=P, g_ik=P, b_ik=P, rope_cos=P, rope_sin=P, kv=P, kv_scale=P, ikv=P, iks=P)
    with pytest.raises(ValueError, match="slot_pos must be 4-byte"):
        _lib.check(_lib.lib().mono_prompt_append_at(C.byref(_lib.PromptAppendArgs(**a)), P + 2, None))


def test_workspaces():
    h = _lib.lib()
    assert h.mono_prompt_attention_workspace(0, 32, 32) == 0 and h.mono_prompt_attention_workspace(100000, 32, 32) == 0
    assert h.mono_prompt_attention_workspace(1, 32, 32) >= 2 * 32 * (512 + 2) * 4
    assert h.mono_prompt_attention_workspace(5, 32, 1) == 0 and h.mono_prompt_attention_workspace(5, 32, 0) == 0
    assert h.mono_prompt_attention_workspace(5, 0, 4) == -1 and b"heads" in h.mono_last_error()
    assert h.mono_prompt_tree_workspace(5, 32, 100) > 0 and h.mono_prompt_tree_workspace(5, 32, -1) == -1


def test_cpu_and_misshapen_tensors_are_refused(monkeypatch):
    bf16, i32, u8 = (dict(dtype=d) for d in (torch.bfloat16, torch.int32, torch.uint8))
    q, at, table = torch.zeros(2, 4, 576, **bf16), torch.zeros(2, **i32), torch.zeros(1, 3, **i32)
    iq, iqs, iw = torch.zeros(2, 64, 64, **u8), torch.zeros(2, 64, 4, **u8), torch.zeros(2, 64, **bf16)
    c = AttnCaches(torch.zeros(5, 4, 64, 16, **u8), torch.zeros(5, 4, 64, **u8), torch.zeros(320, 576, **u8), torch.zeros(320))
    rope, mask = torch.zeros(9, 32), torch.zeros(2, dtype=torch.int64)
    for name, call in (("x", lambda: prompt.index_query(q, at, rope, rope)), ("iq", lambda: prompt.page_scores(iq, iqs, iw, at, at, table, c)),
                       ("scores", lambda: prompt.select_pages(rope, at)), ("q", lambda: prompt.attention(q, at, at, table, table, c)),
                       ("q", lambda: prompt.tree_attention(q, at, at, mask, table, c))):  # fmt: skip
        with pytest.raises(ValueError, match=f"{name}: expected a tensor on a GPU"):
            call()
    monkeypatch.setattr(prompt, "_gpu", lambda t, name: t.device)  # the checks alone, on CPU tensors

    def refused(what, fn, *args, **kw):
        with pytest.raises(ValueError, match=what):
            fn(*args, **kw)

    x = torch.zeros(2, 8192)
    refused("x: expected dtype", prompt.index_query, x.double(), at, rope, rope)
    refused("x: expected shape", prompt.index_query, x[:, :128], at, rope, rope)
    refused("pos: expected dtype", prompt.index_query, x, at.long(), rope, rope)
    refused("rope_cos: expected", prompt.index_query, x, at, rope[:, :8], rope)
    refused("rope_sin", prompt.index_query, x, at, rope, rope[:8])
    refused("iqs", prompt.page_scores, iq, iqs[:1], iw, at, at, table, c)
    refused("iw", prompt.page_scores, iq, iqs, iw.float(), at, at, table, c)
    refused("page_table", prompt.page_scores, iq, iqs, iw, at, at, at, c)
    refused("ikv", prompt.page_scores, iq, iqs, iw, at, at, table, AttnCaches(None, None, None, None))
    refused("columns", prompt.page_scores, iq, iqs, iw, at, at, table, c, columns=-1)
    refused("columns", prompt.page_scores, iq, iqs, iw, at, at, table, c, columns=1 << 32)
    refused("scores: expected", prompt.select_pages, at, at)
    refused("scores: expected dtype", prompt.select_pages, rope.double(), at)
    for kw in (dict(picks=2.0), dict(picks=(1 << 32) + 4), dict(first=-1), dict(last=1 << 32)):
        refused(next(iter(kw)), prompt.select_pages, rope[:2], at, **kw)
    pages = torch.zeros(2, 3, **i32)
    refused("q: expected", prompt.attention, q[..., :512], at, at, pages, table, c)
    refused("q: expected dtype", prompt.attention, q.float(), at, at, pages, table, c)
    refused("q: expected", prompt.attention, q.transpose(0, 1), at, at, pages, table, c)
    refused("pages: expected", prompt.attention, q, at, at, at, table, c)
    refused("pages: expected", prompt.attention, q, at, at, pages.long(), table, c)
    refused("kv: expected", prompt.attention, q, at, at, pages, table, AttnCaches(None, None, None, None))
    refused("kv: expected", prompt.attention, q, at, at, pages, table, AttnCaches(None, None, c.kv[:100], None))
    refused("kv_scale", prompt.attention, q, at, at, pages, table, AttnCaches(None, None, c.kv, c.kv_scale[:64]))
    refused("out", prompt.attention, q, at, at, pages, table, c, out=q)
    refused("starts", prompt.tree_attention, q, at[:1], at[:1], mask, table, c)
    refused("prefix", prompt.tree_attention, q, at, at, mask, table, c)
    refused("mask", prompt.tree_attention, q, at, at[:1], at, table, c)


def test_of_no_columns_no_page_is_selected(monkeypatch):
    """page_scores has no columns where the page table has none (or it is asked for none)."""
    monkeypatch.setattr(prompt, "_gpu", lambda t, name: t.device)
    monkeypatch.setattr(prompt, "_enqueue", lambda dev, fn, args: _lib.check(fn(C.byref(args), None)))
    for tokens in (0, 1, 3):
        got = prompt.select_pages(torch.empty(tokens, 0), torch.arange(tokens, dtype=torch.int32), 5)
        assert got.dtype == torch.int32 and torch.equal(got, torch.full((tokens, 5), -1, dtype=torch.int32))
    for kw in (dict(picks=0), dict(picks=2, first=2, last=1)):
        with pytest.raises(ValueError, match="picks"):
            prompt.select_pages(torch.empty(3, 0), torch.zeros(3, dtype=torch.int32), **kw)


def test_out_over_the_cache_s_scales_is_refused(monkeypatch):
    monkeypatch.setattr(prompt, "_gpu", lambda t, name: t.device)  # the checks alone, on CPU tensors
    at, table, mask = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    q, kv = torch.zeros(2, 4, 576, dtype=torch.bfloat16), torch.zeros(64 * 64, 576, dtype=torch.uint8)
    buf = torch.zeros(4096 + 2048)  # 4096 scales, and behind them as much as an out takes
    c = AttnCaches(None, None, kv, buf[:4096])
    out = buf.view(torch.bfloat16)
    for first in (0, 4096, 8192 - 8):  # the first scales, some in the middle, the last four
        o = out[first:first + 2 * 4 * 512].view(2, 4, 512)
        with pytest.raises(ValueError, match="out: shares memory with kv_scale"):
            prompt.attention(q, at, at, at.view(2, 1), table, c, out=o)
        with pytest.raises(ValueError, match="out: shares memory with kv_scale"):
            prompt.tree_attention(q, torch.zeros(2, dtype=torch.int32), at[:1], mask, table, c, out=o)
    assert prompt._latents(q, c, out[8192:].view(2, 4, 512), q.device)[0] == 64  # right behind them: nothing shared


def test_the_restated_queries_and_scores_are_the_decode_oracle_s():
    torch.manual_seed(5)
    cos, sin = olayer.rope_tables(9)
    x, pos = torch.randn(2, 8192), torch.tensor([3, 8], dtype=torch.int32)
    iq, iqs = ref.index_query(x, pos, cos, sin)
    for n in range(2):
        raw = olayer.codecs.bf16_round(x[n]).view(64, 128)
        rot = torch.cat([olayer.rope_pairs(raw[:, :64], cos[pos[n]], sin[pos[n]]), raw[:, 64:]], -1)
        codes, e8, _, _ = olayer.index_fp4(rot)
        assert float((iq[n] != olayer.codecs.e2m1_pack(codes)).float().mean()) < 1e-2 and torch.equal(iqs[n], e8)
    ikv, iks = torch.randint(0, 256, (4, 4, 64, 16), dtype=torch.uint8), torch.randint(125, 129, (4, 4, 64), dtype=torch.uint8)
    table, iw = torch.tensor([[2, 0, 3]], dtype=torch.int32), torch.randn(2, 64).to(torch.bfloat16)
    at = torch.tensor([150, 64], dtype=torch.int32)
    got, _ = ref.page_scores(iq, iqs, iw, torch.zeros(2, dtype=torch.int32), at, table, ikv, iks, 3)
    keys = oatt.index_scores(iq, iqs, iw, ikv, iks, table.repeat(2, 1), at + 1, 192)
    for n, p in enumerate(at.tolist()):
        for c in range(p // 64 + 1):
            want = keys[n, 64 * c:min(64 * c + 64, p + 1)].max()
            assert abs(float(got[n, c] - want)) <= 1e-4 * max(1.0, abs(float(want)))
        assert bool((got[n, p // 64 + 1:] == -torch.inf).all())


def test_the_restated_attentions_agree():
    """A chain behind a prefix is a token's attention to every page up to its own; the decode
    oracle's over the same slots."""
    torch.manual_seed(6)
    kv = torch.randn(5 * 64, 576).to(torch.float8_e4m3fn).view(torch.uint8)
    scale, table = torch.rand(320) + 0.5, torch.tensor([[3, 1, 4]], dtype=torch.int32)
    q, n = torch.randn(3, 2, 576).to(torch.bfloat16), torch.arange(3, dtype=torch.int32)
    a, _, _ = ref.attention(q, torch.zeros(3, dtype=torch.int32), 100 + n, torch.tensor([[0, 1, 2]] * 3, dtype=torch.int32), table, kv, scale, 0.07)
    b, _, _ = ref.tree_attention(q, torch.tensor([0, 3]), torch.tensor([100]), torch.tensor([1, 3, 7]), table, kv, scale, 0.07)
    sel = torch.full((3, 103), -1, dtype=torch.int32)
    for i in range(3):
        sel[i, :101 + i] = torch.tensor([int(table[0, p // 64]) * 64 + p % 64 for p in range(101 + i)])
    c = oatt.sparse_mla(q, kv, scale, sel, 0.07)
    assert float((a - b).norm() / b.norm()) < 1e-12 and float((a - c).norm() / b.norm()) < 1e-5
