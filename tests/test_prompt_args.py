"""The prompt-width operators' refusals: argument checks run before any GPU call, so they
are testable on the CPU (pointers that no check lets through are never used)."""

import ctypes as C

import pytest
import torch

import prompt_ref as ref
from oracle import layer as olayer
from sgl_amd_mono_amd import _lib, prompt
from sgl_amd_mono_amd.attn import AttnCaches

P = 1 << 20  # an aligned address that is nobody's


def _product(**kw):
    a = dict(x=P, x_stride=256, w=P, s=P, out=P, out_stride=64, out_f32=0, rows=40, n=64, k=256, workspace=P,
             workspace_bytes=1 << 20)
    a.update(kw)
    return _lib.lib().mono_prompt_product(C.byref(_lib.PromptProductArgs(**a)), None)


@pytest.mark.parametrize("kw,what", [
    (dict(rows=-1), "rows"), (dict(rows=(1 << 20) + 1), "rows"), (dict(n=24), "n must"), (dict(n=0), "n must"),
    (dict(n=1 << 20), "n must"), (dict(k=192), "k must"), (dict(k=0), "k must"), (dict(x=None), "x must"),
    (dict(x=P + 8), "x must be 16-byte"), (dict(w=None), "w must"), (dict(s=None), "s must"), (dict(out=None), "out must"),
    (dict(x_stride=255), "x_stride"), (dict(x_stride=128), "x_stride"), (dict(out_stride=60), "out_stride"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=100), "workspace must hold"), (dict(workspace=P + 16), "workspace"),
    (dict(rows=1 << 20, k=1 << 15), "rows x k must be at most 34359738367"),
])  # fmt: skip
def test_product_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _lib.check(_product(**kw))


def test_product_of_no_rows_looks_at_nothing():
    _lib.check(_product(rows=0, x=None, w=None, s=None, out=None, workspace=None, workspace_bytes=0))


def test_workspaces():
    h = _lib.lib()
    assert h.mono_prompt_product_workspace(40, 64, 256) >= 40 * 256 + 40 * 2 * 4
    assert h.mono_prompt_product_workspace(5, 64, 256) == 0  # few rows need none
    assert h.mono_prompt_product_workspace(0, 64, 256) == 0
    assert h.mono_prompt_product_workspace(5, 60, 256) == -1 and b"n must" in h.mono_last_error()
    a = _lib.PromptExpertsArgs(tokens=10, picks=2, experts=4, shared=1, hidden=256, inter=128)
    assert h.mono_prompt_experts_workspace(C.byref(a)) > 0
    a.experts = 0
    assert h.mono_prompt_experts_workspace(C.byref(a)) == -1


def _append(**kw):
    a = dict(kv_a=P, kv_stride=576, ik=P, ik_stride=128, f32=0, tokens=3, req=P, pos=P, page_table=P, requests=2,
             pt_stride=4, n_pages=8, max_pos=100, g_kv=P, g_ik=P, b_ik=P, rope_cos=P, rope_sin=P, kv=P, kv_scale=P, ikv=P,
             iks=P)
    a.update(kw)
    return _lib.lib().mono_prompt_append(C.byref(_lib.PromptAppendArgs(**a)), None)


@pytest.mark.parametrize("kw,what", [
    (dict(tokens=-1), "tokens"), (dict(requests=-1), "requests"), (dict(max_pos=-1), "max_pos"), (dict(kv_stride=572), "kv_stride"),
    (dict(kv_stride=570, f32=1), "kv_stride"), (dict(ik_stride=129), "ik_stride"), (dict(kv_a=P + 4), "kv_a"),
    (dict(ik=P + 4), "ik must"), (dict(req=None), "req"), (dict(pos=None), "pos"), (dict(page_table=None), "page_table"),
    (dict(g_kv=None), "g_kv"), (dict(rope_sin=None), "rope_sin"), (dict(kv=None), "kv must"), (dict(ikv=None), "ikv"),
    (dict(iks=None), "iks"),
])  # fmt: skip
def test_append_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _lib.check(_append(**kw))


def _experts(**kw):
    a = dict(x=P, x_stride=256, ids=P, weights=P, w13=P, s13=P, w2=P, s2=P, residual=P, residual_stride=256, out=P,
             out_stride=256, tokens=4, picks=2, experts=8, shared=1, hidden=256, inter=128, workspace=P,
             workspace_bytes=1 << 24)
    a.update(kw)
    return _lib.lib().mono_prompt_experts(C.byref(_lib.PromptExpertsArgs(**a)), None)


@pytest.mark.parametrize("kw,what", [
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 20), "tokens x"), (dict(picks=0), "picks"), (dict(picks=65), "picks"),
    (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(hidden=200), "hidden"), (dict(inter=64), "inter"),
    (dict(x_stride=250), "x_stride"), (dict(residual_stride=128), "residual_stride"), (dict(residual=P + 2), "residual"),
    (dict(ids=None), "ids"), (dict(weights=None), "weights"), (dict(w13=None), "w13"), (dict(s2=None), "s2"),
    (dict(out=P + 8), "out must"), (dict(workspace_bytes=0), "workspace"),
    (dict(tokens=1 << 19, picks=1, hidden=1 << 16), "tokens x hidden"),
])  # fmt: skip
def test_experts_refusals(kw, what):
    with pytest.raises(ValueError, match=what):
        _lib.check(_experts(**kw))


def test_null_args():
    h = _lib.lib()
    for fn in (h.mono_prompt_product, h.mono_prompt_append, h.mono_prompt_experts):
        with pytest.raises(ValueError, match="args is NULL"):
            _lib.check(fn(None, None))


def test_cpu_tensors_are_refused():
    x, w, s = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(16, 128, dtype=torch.uint8), torch.zeros(1, 1)
    with pytest.raises(ValueError, match="x: expected a tensor on a GPU"):
        prompt.product(x, w, s)
    with pytest.raises(ValueError, match="x: expected a tensor"):
        prompt.experts([1], w, s, w, s, w, s)
    with pytest.raises(ValueError, match="kv_a: expected a tensor on a GPU"):
        prompt.append(x, x, s, s, s, AttnCaches(w, w, w, None), s, s, s, s, s)


def test_what_is_no_tensor_is_refused_by_name(monkeypatch):
    monkeypatch.setattr(prompt, "_gpu", lambda t, name: t.device)  # the checks alone, on CPU tensors
    bf16, f32, i32 = (dict(dtype=d) for d in (torch.bfloat16, torch.float32, torch.int32))
    x, w, s = torch.zeros(2, 128, **bf16), torch.zeros(16, 128, dtype=torch.uint8), torch.zeros(1, 1)
    for out in ([0], 1.5, "out"):
        with pytest.raises(ValueError, match="out: expected a tensor"):
            prompt.product(x, w, s, out=out)
    kv_a, ik, at, table = torch.zeros(2, 576, **bf16), torch.zeros(2, 128, **bf16), torch.zeros(2, **i32), torch.zeros(1, 1, **i32)
    rest = (torch.zeros(512, **bf16), torch.zeros(128, **f32), torch.zeros(128, **f32), torch.zeros(9, 32), torch.zeros(9, 32))
    for ikv in (None, [1], torch.tensor(3)):
        with pytest.raises(ValueError, match="ikv: expected"):
            prompt.append(kv_a, ik, at, at, table, AttnCaches(ikv, w, w, None), *rest)


def test_shared_memory_is_told_apart():
    wide = torch.zeros(6, 64, dtype=torch.bfloat16)
    a, b = wide[:, :32], wide[:, 32:]
    assert prompt._apart(a, 64, b, 64) and prompt._apart(b, 64, a, 64)
    assert not prompt._apart(a, 64, wide[:, 24:48], 64) and not prompt._apart(wide[:, 24:48], 64, a, 64)
    assert not prompt._apart(a, 64, a, 64)
    assert prompt._apart(wide[:2], 64, wide[2:], 64) and not prompt._apart(wide[:3], 64, wide[2:], 64)
    assert not prompt._apart(a, 64, wide.view(12, 32)[::2][:, :16], 32)  # other strides: only ranges are told apart
    assert prompt._apart(a[:0], 64, a, 64)


def test_the_restated_append_is_the_front_s_row():
    """The f64 restatement writes what the decode layer's oracle (f32) writes, on values
    where no code hangs on f32's last bits."""
    torch.manual_seed(3)
    n = 3
    kv_a, ik = torch.randn(n, 576), torch.randn(n, 128)
    g_kv, g_ik, b_ik = torch.ones(512), torch.ones(128), torch.zeros(128)
    cos, sin = olayer.rope_tables(16)
    pos = torch.arange(n, dtype=torch.int32)
    caches = dict(ikv=torch.zeros(1, 4, 64, 16, dtype=torch.uint8), iks=torch.zeros(1, 4, 64, dtype=torch.uint8),
                  kv=torch.zeros(64, 576, dtype=torch.uint8), kv_scale=torch.zeros(64))
    ref.append(kv_a, ik, torch.zeros(n, dtype=torch.int32), pos, torch.zeros(1, 1, dtype=torch.int32), caches, g_kv, g_ik,
               b_ik, cos, sin)
    kvn = olayer.codecs.bf16_round(olayer.rmsnorm(kv_a[:, :512], g_kv))
    kpe = olayer.codecs.bf16_round(olayer.rope_pairs(kv_a[:, 512:], cos[:n], sin[:n]))
    codes, scale = olayer.fp8_row_quant_pow2(torch.cat([kvn, kpe], -1))
    k_codes, k_e8, _, _ = olayer.index_key(ik, g_ik, b_ik, cos[:n], sin[:n])
    assert float((caches["kv"][:n] != codes).float().mean()) < 1e-2 and torch.equal(caches["kv_scale"][:n], scale)
    got = caches["ikv"][0, :, :n].transpose(0, 1).reshape(n, 64)
    assert float((got != olayer.codecs.e2m1_pack(k_codes)).float().mean()) < 2e-2
    assert torch.equal(caches["iks"][0, :, [0, 4, 8]].T, k_e8)
