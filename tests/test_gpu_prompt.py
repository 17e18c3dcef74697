"""The prompt-width operators on the GPU against their float64 restatements.

Tolerances, from the formats. A bf16 output is off by half a step, 2^-8 of it. The FP8
MFMA adds a block's 128 products with fewer bits than f32's (1.4e-5 of the result on
N(0, 1) values): 2^-14 of the sum of the terms' magnitudes holds some thirty times that.
An f32 product's K sums are each off by at most 2^-24 of what has been summed. Rows in
bf16 have no code that hangs on a rounding (a quotient that is a tie is one exactly), a
mid may: an error of 2^-14 moves at most 2^-9 of the mids (2^-14 of the distance 2^-4
between borders, both sides) over one, each by 2^-3 of itself, so the sums by
2^-3 sqrt(2^-9) < 0.0056 of their size. One output may lie further off: a single mid that
moves by a code moves it by that step times a weight, whatever the sums' size, so two such
steps are allowed in each of a token's experts (prompt_ref.experts' ``step``).
Appended rows are formed in f64 on both sides: they are equal.
"""

import pytest
import torch

import prompt_ref as ref
from oracle import attention as oatt
from oracle import codecs
from oracle import layer as olayer
from sgl_amd_mono_amd import prompt, workloads
from sgl_amd_mono_amd.attn import AttnCaches, AttnRuntime, AttnStep
from sgl_amd_mono_amd.layer import KV_LORA, N_QKV, PE_DIM, Q_LORA, ProjRuntime
from sgl_amd_mono_amd.layouts import shuffle_16x16
from sgl_amd_mono_amd.moe import FP8_MOE, MoeGeometry, MoeRuntime

pytestmark = pytest.mark.gpu


def _matrix(n, k, dev, seed):
    return workloads._fp8_matrix(n, k, torch.Generator(device=dev).manual_seed(seed), dev)


def _same(got, want, mag, f32, k):
    """Within the tolerances of the module's head."""
    # a sum past the type's largest value is its infinity, as the rounding of that sum is
    far = want.abs() > torch.finfo(got.dtype).max
    got, bad = got.cpu().double(), want.isnan()
    assert bool((got.isnan() == bad).all()) and torch.equal(got[far], torch.inf * want[far].sign())
    bad = bad | far
    tol = k * 2.0**-24 * mag + 2.0**-24 * want.abs() if f32 else 2.0**-8 * want.abs() + 2.0**-14 * mag
    over = ((got - want).abs() / tol.clamp_min(1e-30))[~bad]
    assert float(over.max() if over.numel() else 0.0) <= 1.0, float(over.max())


# ------------------------------------------------------------------- product
@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (1, 2112, 7168), (3, 144, 384), (16, 128, 7168), (17, 272, 1024),
                                   (63, 64, 256), (65, 2112, 512), (129, 400, 1152), (300, 1536, 640),
                                   # the borders of each way to run: few rows, K shared out, tiles of 64 and 128 rows
                                   (16, 64, 2048), (17, 64, 2048), (16, 64, 2176), (4, 32, 8192), (5, 32, 8192), (45, 144, 7168),
                                   (96, 16, 4096), (97, 16, 4096), (300, 528, 4096), (2050, 4112, 256), (4100, 16, 128)])
def test_product(gpu_device, m, n, k, f32):
    w, s = _matrix(n, k, gpu_device, 1)
    x = workloads.rows_bf16(m, k, gpu_device, seed=2)
    x[0, : k // 2] *= 100.0  # blocks of other sizes next to each other
    got = prompt.product(x, w, s, dtype=torch.float32 if f32 else torch.bfloat16)
    want, mag = ref.product(x.cpu(), w.cpu(), s.cpu())
    _same(got, want, mag, f32, k)


@pytest.mark.parametrize("m,n,k", [(5, 64, 2048), (16, 2112, 2048),  # few rows, rounded in the workgroup
                                   (20, 256, 640), (100, 64, 640), (45, 128, 7168), (96, 16, 4096),  # narrow; K shared out
                                   (300, 1536, 640), (1025, 528, 1024), (300, 528, 4096), (200, 2112, 7168)])  # wide; shared out
def test_product_f32_sums(gpu_device, m, n, k):
    """The sums of an f32 product are f32's. A running sum over kb blocks is rounded kb times,
    2^-24 of what it then is: sqrt(kb / 2) 2^-24 of the result in the mean, as the parts of a
    sum of independent terms grow; the block's scales, its product's four steps and eight
    waves' sums are 10 roundings at most of all of it: at kb = 56 within 16 x 2^-24 = 9.5e-7
    of the norm. The FP8 MFMA's own sums are 1.4e-5 off."""
    w, s = _matrix(n, k, gpu_device, 18)
    x = workloads.rows_bf16(m, k, gpu_device, seed=19)
    got = prompt.product(x, w, s, dtype=torch.float32).cpu().double()
    want, _ = ref.product(x.cpu(), w.cpu(), s.cpu())
    off = float((got - want).norm() / want.norm())
    print(f"{off:.2e}", flush=True)
    assert off <= 16 * 2.0**-24


@pytest.mark.parametrize("m", [1, 15, 64, 200, 257, 530, 1025])
@pytest.mark.parametrize("n", [16, 208, 256, 528])
def test_product_of_small_integers_is_exact(gpu_device, m, n):
    """Integers within a factor of 7 of each other: every code, product and sum is exact,
    so a wrong place anywhere shows."""
    k = 512
    g = torch.Generator(device=gpu_device).manual_seed(m * n)
    x = torch.randint(-7, 8, (m, k), generator=g, device=gpu_device).float()
    x[:, ::128] = 7.0  # each block's scale is 7 / 448 = 1 / 64
    w = torch.randint(-4, 5, (n, k), generator=g, device=gpu_device).float()
    s = 2.0 ** torch.randint(-2, 3, (-(-n // 128), k // 128), generator=g, device=gpu_device).float()
    got = prompt.product(x.to(torch.bfloat16), shuffle_16x16(w.to(torch.float8_e4m3fn)), s, dtype=torch.float32)
    full = (w * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)).double()
    assert torch.equal(got.cpu().double(), x.cpu().double() @ full.cpu().T)


@pytest.mark.parametrize("m", [9, 30, 77, 200, 4500])
def test_product_strided_rows_and_out(gpu_device, m):
    n, k = 2112 if m > 4000 else 192, 384  # (4500 rows: tiles of 128)
    w, s = _matrix(n, k, gpu_device, 3)
    wide = workloads.rows_bf16(m, k + 64, gpu_device, seed=4)
    buf = torch.full((m + 2, n + 48), 3.0, dtype=torch.bfloat16, device=gpu_device)  # what lies around out stays
    got = prompt.product(wide[:, 64:], w, s, out=buf[1:-1, 16:-32])
    assert torch.equal(got, prompt.product(wide[:, 64:].contiguous(), w, s))
    assert bool((buf[0] == 3).all()) and bool((buf[-1] == 3).all())
    assert bool((buf[:, :16] == 3).all()) and bool((buf[:, -32:] == 3).all())


@pytest.mark.parametrize("m", [5, 70, 300])
def test_product_non_finite_and_extreme_rows(gpu_device, m):
    n, k = 64, 512
    w, s = _matrix(n, k, gpu_device, 5)
    x = workloads.rows_bf16(m, k, gpu_device, seed=6)
    x[1, 130] = float("nan")
    x[2, 511] = float("-inf")
    x[3] = 0.0
    x[4, :128] = torch.finfo(torch.bfloat16).max
    x[4, 128:256] = 1e-39  # below the least block size
    got = prompt.product(x, w, s, dtype=torch.float32)
    want, mag = ref.product(x.cpu(), w.cpu(), s.cpu())
    assert bool(got[1:3].isnan().all()) and bool((got[3] == 0).all())
    _same(got, want, mag, True, k)


@pytest.mark.parametrize("m", [3, 30, 200])
def test_product_nan_weights_stay_in_their_output(gpu_device, m):
    n, k = 80, 1280
    w, s = _matrix(n, k, gpu_device, 8)
    x = workloads.rows_bf16(m, k, gpu_device, seed=9)
    clean = prompt.product(x, w, s)
    flat = w.view(torch.uint8).flatten()  # row 37, column 1279 in the (16, 16) layout
    flat[((37 // 16 * (k // 32) + 1279 // 32) * 2 + 1279 % 32 // 16) * 256 + 37 % 16 * 16 + 1279 % 16] = 0x7F
    got = prompt.product(x, w, s)
    assert bool(got[:, 37].isnan().all())
    keep = [c for c in range(n) if c != 37]
    assert torch.equal(got[:, keep], clean[:, keep])


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("m,k", [(3, 1280), (30, 1280), (30, 2304), (200, 1280)])
def test_product_infinite_weight_scale(gpu_device, m, k, f32):
    """A weight block whose scale is infinite makes its outputs infinite, with the sign of the
    block's own sum, whichever way the product runs."""
    n = 80
    w, s = _matrix(n, k, gpu_device, 14)
    x = workloads.rows_bf16(m, k, gpu_device, seed=15)
    first = ref.rounded(x[:, :128].cpu()) @ ref.weight(w.cpu(), s.cpu())[:, :128].T
    s[0, 0] = float("inf")
    got = prompt.product(x, w, s, dtype=torch.float32 if f32 else torch.bfloat16).cpu().double()
    clear = first.abs() > 2.0**-14 * 8.0 * first.abs().max()  # its sign hangs on no rounding of the block's sum
    assert bool(got.isinf().all()) and torch.equal(got.sign()[clear], first.sign()[clear])
    assert float(clear.float().mean()) > 0.9


@pytest.mark.parametrize("m,stride", [(5, 1 << 29), (40, 1 << 26), (300, 1 << 23)])
def test_product_rows_far_apart(gpu_device, m, stride):
    """Row offsets past 32 bits."""
    n, k = 64, 256
    w, s = _matrix(n, k, gpu_device, 10)
    x = workloads.rows_bf16(m, k, gpu_device, seed=11)
    far = torch.empty((m - 1) * stride + k, dtype=torch.bfloat16, device=gpu_device).as_strided((m, k), (stride, 1))
    far.copy_(x)
    assert torch.equal(prompt.product(far, w, s), prompt.product(x, w, s))


def test_product_of_the_most_elements(gpu_device):
    """As many elements as a call takes: their rounding needs more threads than one launch has
    (rows around the borders of its launches, 262656 rows each, against 64 bits)."""
    n, m, k = 16, 525314, 65408
    torch.cuda.empty_cache()
    w, s = _matrix(n, k, gpu_device, 16)
    x = torch.empty(m, k, dtype=torch.bfloat16, device=gpu_device)  # (what lies in the other rows is theirs)
    at = [0, 1, 262655, 262656, 393985, 525311, 525312, 525313]
    x[at] = workloads.rows_bf16(len(at), k, gpu_device, seed=17)
    got = prompt.product(x, w, s)[at]
    x = x[at].cpu()
    torch.cuda.empty_cache()
    _same(got, *ref.product(x, w.cpu(), s.cpu()), False, k)


def test_product_refuses_shared_memory(gpu_device):
    w, s = _matrix(256, 256, gpu_device, 12)
    x = workloads.rows_bf16(4, 512, gpu_device, seed=13)
    want = prompt.product(x[:, :256].clone(), w, s)
    with pytest.raises(ValueError, match="shares memory with x"):
        prompt.product(x[:, :256], w, s, out=x[:, :256])
    assert torch.equal(prompt.product(x[:, :256], w, s, out=x[:, 256:]), want)


def test_product_of_no_rows(gpu_device):
    w, s = _matrix(64, 256, gpu_device, 7)
    assert prompt.product(torch.empty(0, 256, dtype=torch.bfloat16, device=gpu_device), w, s).shape == (0, 64)


# -------------------------------------------------------------------- append
def _append_case(dev, spans, f32, raw, pads=0, wide=0, seed=11):
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-(a + n) // 64) for a, n in spans]
    pages, width = sum(need) + 3, max(need) + 1
    table = torch.zeros(len(spans), width, dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    at = 0
    for r, u in enumerate(need):
        table[r, :u] = order[at:at + u]
        at += u
    req = torch.cat([torch.full((n,), r) for r, (_, n) in enumerate(spans)] + [torch.full((pads,), -1)]).int()
    pos = torch.cat([torch.arange(a, a + n) for a, n in spans] + [torch.zeros(pads)]).int()
    t, dt = len(req), torch.float32 if f32 else torch.bfloat16
    kv_a = (2.0 * torch.randn(t, 576 + wide, generator=g, device=dev)).to(dt)[:, wide:]
    ik = (torch.randn(t, 128 + wide, generator=g, device=dev) + 0.2).to(dt)[:, wide:]
    u8 = dict(generator=g, device=dev, dtype=torch.uint8)
    caches = AttnCaches(ikv=torch.randint(0, 256, (pages, 4, 64, 16), **u8), iks=torch.randint(120, 130, (pages, 4, 64), **u8),
                        kv=torch.randint(0, 126, (pages * 64, 576), **u8),
                        kv_scale=None if raw else torch.rand(pages * 64, generator=g, device=dev))
    cos, sin = workloads.rope_tables(width * 64 - 5, dev)
    w = dict(g_kv=(1 + 0.1 * torch.randn(512, generator=g, device=dev)).to(torch.bfloat16),
             g_ik=1 + 0.1 * torch.randn(128, generator=g, device=dev), b_ik=0.1 * torch.randn(128, generator=g, device=dev))
    return dict(kv_a=kv_a, ik=ik, req=req.to(dev), pos=pos.to(dev), page_table=table.to(dev), caches=caches, **w,
                rope_cos=cos, rope_sin=sin)


def _append_both(c):
    """Run the operator on c's caches; returns (what it left, what it should leave)."""
    want = {k: None if v is None else v.cpu().clone() for k, v in vars(c["caches"]).items()}
    cpu = {k: v.cpu() for k, v in c.items() if k != "caches"}
    ref.append(cpu["kv_a"], cpu["ik"], cpu["req"], cpu["pos"], cpu["page_table"], want, cpu["g_kv"], cpu["g_ik"],
               cpu["b_ik"], cpu["rope_cos"], cpu["rope_sin"])
    prompt.append(**c)
    return {k: None if v is None else v.cpu() for k, v in vars(c["caches"]).items()}, want


def _equal(got, want):
    for k, v in want.items():
        assert (v is None and got[k] is None) or torch.equal(got[k], v), k


@pytest.mark.parametrize("f32", [False, True], ids=["bf16", "f32"])
@pytest.mark.parametrize("raw", [False, True], ids=["scaled", "raw"])
@pytest.mark.parametrize("spans,pads,wide", [([(0, 1)], 0, 0), ([(700, 1), (63, 1), (64, 1)], 2, 0),
                                             ([(0, 64), (60, 9), (1, 130)], 5, 16), ([(0, 333)], 0, 1536)])
def test_append(gpu_device, spans, pads, wide, f32, raw):
    _equal(*_append_both(_append_case(gpu_device, spans, f32, raw, pads, wide)))


def test_append_out_of_range_tokens_write_nothing(gpu_device):
    c = _append_case(gpu_device, [(0, 70), (10, 60)], False, False, pads=4)
    pages = c["caches"].ikv.shape[0]
    c["req"][3], c["req"][4] = 2, -7  # no such request
    c["pos"][5], c["pos"][6] = -1, 1 << 30  # no such position
    c["pos"][7] = c["rope_cos"].shape[0]  # no angle
    c["page_table"][1, 0] = pages  # bad pages
    c["page_table"][0, 1] = -1
    _equal(*_append_both(c))


def test_append_extreme_rows(gpu_device):
    c = _append_case(gpu_device, [(0, 12)], True, False)
    c["kv_a"][0] = 0.0
    c["ik"][0] = 0.0
    c["kv_a"][1] = 1e-30
    c["ik"][1] = 5.0  # no variance: the bias alone
    c["kv_a"][2, :512] *= 1e18
    c["kv_a"][3, 512:] = 1e6
    c["kv_a"][4, 512:] = 448.0 * 2.0**-3  # an amax that is exactly a scale's border, before rotation
    c["pos"][4] = 0
    c["pos"][0] = 4
    _equal(*_append_both(c))


@pytest.mark.parametrize("raw", [False, True], ids=["scaled", "raw"])
def test_append_non_finite(gpu_device, raw):
    """A NaN stays a NaN that a reader sees, and stays in its own token."""
    c = _append_case(gpu_device, [(0, 8)], False, raw)
    clean = _append_case(gpu_device, [(0, 8)], False, raw)
    c["kv_a"][2, 5] = float("nan")
    c["ik"][3, 9] = float("inf")
    prompt.append(**c)
    prompt.append(**clean)
    got, want = c["caches"], clean["caches"]
    page = int(c["page_table"][0, 0])
    assert bool(((got.kv[page * 64 + 2, :512] & 0x7F) == 0x7F).all())
    assert bool((got.iks[page, :, 3 * 4] == 255).all())
    others = [t for t in range(64) if t != 2]
    assert torch.equal(got.kv.view(-1, 64, 576)[page, others], want.kv.view(-1, 64, 576)[page, others])
    others = [t for t in range(64) if t != 3]
    assert torch.equal(got.ikv[page, :, others], want.ikv[page, :, others])


def test_append_far_into_a_long_cache(gpu_device):
    """Slots whose rows lie past 2^31 bytes."""
    c = _append_case(gpu_device, [(60, 9)], False, False)
    want, _ = _append_both(c)
    pages, near = 60000, c["page_table"][0].tolist()
    far = dict(c, page_table=c["page_table"] + (pages - 8))
    big = AttnCaches(ikv=torch.empty(pages, 4, 64, 16, dtype=torch.uint8, device=gpu_device),
                     iks=torch.empty(pages, 4, 64, dtype=torch.uint8, device=gpu_device),
                     kv=torch.empty(pages * 64, 576, dtype=torch.uint8, device=gpu_device),
                     kv_scale=torch.empty(pages * 64, device=gpu_device))
    prompt.append(**dict(far, caches=big))
    for p in (60, 63, 64, 68):
        a, b, t = near[p // 64], near[p // 64] + pages - 8, p % 64
        assert torch.equal(big.kv[b * 64 + t].cpu(), want["kv"][a * 64 + t])
        assert float(big.kv_scale[b * 64 + t]) == float(want["kv_scale"][a * 64 + t])
        assert torch.equal(big.ikv[b, :, t].cpu(), want["ikv"][a, :, t])
        at = t % 16 * 4 + t // 16
        assert torch.equal(big.iks[b, :, at].cpu(), want["iks"][a, :, at])


def test_append_of_nothing(gpu_device):
    c = _append_case(gpu_device, [(0, 3)], False, False)
    before = c["caches"].kv.clone()
    for k in ("kv_a", "ik", "req", "pos"):
        c[k] = c[k][:0]
    prompt.append(**c)
    assert torch.equal(c["caches"].kv, before)


# ------------------------------------------------------------------- experts
def _experts_case(dev, t, h, i, e, k, seed=21, shared=True):
    geo = MoeGeometry(h, e, k, i, 1.0, 1e-6, "sigmoid_bias", "fp8_block128")
    m = workloads.fp8_moe_weights(geo, dev, seed=seed)
    m.s13 *= 448.0 / (1.25 * h**0.5)
    m.s2 *= 448.0 / (1.25 * i**0.5)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    ids = torch.rand(t, e, generator=g, device=dev).argsort(1)[:, :k].int().contiguous()
    wts = torch.rand(t, k, generator=g, device=dev) + 0.1
    x = workloads.rows_bf16(t, h, dev, seed=seed + 2)
    n = e + 1 if shared else e
    return dict(x=x, ids=ids, weights=wts, w13=m.w13[:n].contiguous(), s13=m.s13[:n].contiguous(), w2=m.w2[:n].contiguous(),
                s2=m.s2[:n].contiguous(), residual=workloads.rows_bf16(t, h, dev, seed=seed + 3), shared=shared)


def _check_experts(c, got):
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    want, y, step = ref.experts(cpu["x"], cpu["ids"], cpu["weights"], cpu["w13"], cpu["s13"], cpu["w2"], cpu["s2"],
                                cpu["residual"], cpu["shared"])
    d = got.cpu().double() - want
    assert not bool(d.isnan().any())
    over = d.abs() / (2.0**-8 * want.abs() + 2 * step[:, None] + 1e-30)
    assert float(over.max()) <= 1.0, float(over.max())
    assert float(d.norm()) <= 0.0056 * float(y.norm()) + 2.0**-8 * float(want.norm())


@pytest.mark.parametrize("t,h,i,e,k", [(1, 256, 128, 4, 1), (1, 512, 256, 16, 8), (9, 384, 128, 5, 5), (40, 256, 384, 8, 2),
                                       (130, 512, 128, 3, 2), (300, 256, 256, 33, 4), (700, 128, 128, 2, 1),
                                       # wide and narrow tiles over every number of mid blocks up to one too many for LDS
                                       (200, 384, 384, 4, 2), (150, 128, 512, 5, 2), (150, 1152, 640, 3, 2), (30, 384, 512, 4, 3),
                                       (30, 128, 640, 4, 3), (3, 640, 768, 9, 2),
                                       # as many experts and picks as a call takes, narrow and wide
                                       (9, 128, 128, 1024, 64), (150, 128, 128, 1024, 64), (200, 128, 128, 1024, 64)])
def test_experts(gpu_device, t, h, i, e, k):
    c = _experts_case(gpu_device, t, h, i, e, k)
    _check_experts(c, prompt.experts(**c))


def test_experts_without_shared_or_residual(gpu_device):
    c = _experts_case(gpu_device, 50, 256, 128, 8, 2, shared=False)
    got = prompt.experts(**dict(c, residual=None))
    c["residual"] = torch.zeros_like(c["x"])
    _check_experts(c, got)


@pytest.mark.parametrize("t,h,i,e,k", [(150, 1152, 128, 3, 2), (130, 2048, 256, 2, 1), (150, 2432, 384, 3, 2), (300, 7168, 512, 4, 2)])
def test_experts_wide_columns(gpu_device, t, h, i, e, k):
    """Wide calls whose mids stay in LDS over more columns than one workgroup takes: even and
    uneven turns of columns, the last past the matrix, tiles of more rows than 64 and of fewer."""
    c = _experts_case(gpu_device, t, h, i, e, k)
    few = torch.rand(t, generator=torch.Generator().manual_seed(t)).to(gpu_device) < 0.2
    c["ids"][:, 0] = torch.where(few, e - 1, 0).int()  # the last expert gets some, the first most
    if k > 1:
        c["ids"][:, 1] = 1
    _check_experts(c, prompt.experts(**c))


@pytest.mark.parametrize("invariant", [False, True])
def test_experts_narrow_up_products_are_exact(gpu_device, invariant):
    """Beside its own rounding to bf16, an output of the narrow tiles is off by the parts' f16
    (2^-11 / sqrt(3) = 0.00028 of the norm) and by mids over a border: one that is 1e-6 off (f32
    sums, a few last bits of the SiLU) crosses with the probability 1e-6 / step and moves by a
    step of at most 2^-3 of itself, sqrt(1e-6 x 2^-3) = 0.00036 of the norm; together 0.00046.
    The FP8 MFMA's 1.4e-5 makes it 0.001."""
    t = 300 if invariant else 64
    c = dict(_experts_case(gpu_device, t, 1024, 512, 2, 1, shared=False), residual=None)
    c["weights"][:] = 1.0
    got = prompt.experts(**c, batch_invariant=invariant).cpu().double()
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    want, _, _ = ref.experts(cpu["x"], cpu["ids"], cpu["weights"], cpu["w13"], cpu["s13"], cpu["w2"], cpu["s2"], shared=False)
    own = want.float().to(torch.bfloat16).double() - want
    off = float(((got - want).square().sum() - own.square().sum()).clamp_min(0).sqrt() / want.norm())
    print(f"{off:.2e}", flush=True)
    assert off <= 0.00046


@pytest.mark.parametrize("t", [6, 90, 400])
def test_experts_odd_picks(gpu_device, t):
    """Picks of no expert, tokens without any, one expert twice, an expert that all pick."""
    c = _experts_case(gpu_device, t, 256, 128, 8, 4)
    c["ids"][:, 0] = 5
    c["ids"][1] = -1
    c["ids"][2, 1:] = torch.tensor([8, 9, 1 << 30], device=gpu_device).int()  # 8 is the shared one: not a pick
    c["ids"][3] = torch.tensor([2, 2, 2, 6], device=gpu_device).int()
    c["weights"][1] = float("nan")  # the weight of no pick
    _check_experts(dict(c, weights=c["weights"].nan_to_num(0.0)), prompt.experts(**c))
    c["ids"][:] = -1  # no pick at all: the shared expert alone
    c["weights"][1] = 1.0
    _check_experts(c, prompt.experts(**c))
    c = dict(_experts_case(gpu_device, t, 256, 128, 8, 4, shared=False), residual=None)
    c["ids"][:] = 8
    assert bool((prompt.experts(**c) == 0).all())


@pytest.mark.parametrize("counts", [(16, 17, 1, 30), (32, 33, 0, 64), (65, 1, 0, 62), (128, 129, 64, 65), (256, 0, 1, 257)])
def test_experts_tile_borders(gpu_device, counts):
    """Experts whose rows end on, before and behind a tile's last one, and experts without any."""
    t = sum(counts)
    c = _experts_case(gpu_device, t, 256, 128, len(counts), 1)
    order = torch.randperm(t, generator=torch.Generator().manual_seed(t)).to(gpu_device)
    c["ids"] = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)]).int().to(gpu_device)[order][:, None].contiguous()
    _check_experts(c, prompt.experts(**c))


@pytest.mark.parametrize("t", [33, 500])
def test_experts_ids_anywhere(gpu_device, t):
    """Ids and weights that are contiguous and lie at any element (not 16-byte aligned)."""
    c = _experts_case(gpu_device, t, 256, 128, 8, 3)
    want = prompt.experts(**c)
    for off in (1, 2, 3):
        ids = torch.zeros(t * 3 + 4, dtype=torch.int32, device=gpu_device)[off:off + t * 3].view(t, 3)
        wts = torch.zeros(t * 3 + 4, device=gpu_device)[off:off + t * 3].view(t, 3)
        assert torch.equal(prompt.experts(**dict(c, ids=ids.copy_(c["ids"]), weights=wts.copy_(c["weights"]))), want)


def test_experts_strided_in_place(gpu_device):
    c = _experts_case(gpu_device, 33, 256, 128, 8, 2)
    want = prompt.experts(**c)
    buf = torch.zeros(33, 256 + 40, dtype=torch.bfloat16, device=gpu_device)
    buf[:, 8:-32] = c["residual"]
    xw = torch.zeros(33, 256 + 8, dtype=torch.bfloat16, device=gpu_device)
    xw[:, 8:] = c["x"]
    got = prompt.experts(**dict(c, x=xw[:, 8:], residual=buf[:, 8:-32], out=buf[:, 8:-32]))
    assert torch.equal(got, want) and bool((buf[:, :8] == 0).all()) and bool((buf[:, -32:] == 0).all())


def test_experts_out_over_x_and_residual(gpu_device):
    c = _experts_case(gpu_device, 200, 256, 128, 8, 2)
    want = prompt.experts(**c)
    x = c["x"].clone()
    assert torch.equal(prompt.experts(**dict(c, x=x, out=x)), want)
    res = torch.cat([c["residual"], c["residual"][:1]])
    with pytest.raises(ValueError, match="shares memory with residual"):
        prompt.experts(**dict(c, residual=res[:-1], out=res[1:]))
    assert torch.equal(prompt.experts(**dict(c, residual=res[:-1], out=res[:-1])), want)


def test_experts_non_finite_tokens(gpu_device):
    """A token's NaN or infinity is its own: the others' outputs keep their bits."""
    for t in (20, 200):
        c = _experts_case(gpu_device, t, 256, 128, 8, 2)
        want = prompt.experts(**c)
        x = c["x"].clone()
        x[3, 7], x[5, 200] = float("nan"), float("inf")
        got = prompt.experts(**dict(c, x=x))
        assert bool(got[3].isnan().all()) and bool(got[5].isnan().all())
        keep = [i for i in range(t) if i not in (3, 5)]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("t,h,i", [(20, 256, 128), (200, 256, 128), (20, 384, 640), (200, 384, 640)])
def test_experts_infinite_sum_leaves_its_neighbours(gpu_device, t, h, i):
    """A down product past f32's range is an infinity in its own column: the other columns,
    far above f16's largest value, keep the bits that they have where that column's weights
    are zero (narrow and wide tiles, mids in LDS and not)."""
    c = _experts_case(gpu_device, t, h, i, 8, 2)
    c["s2"] *= 2.0**122
    clean, col = {}, 70
    for code, to in ((0x7E, c), (0x00, clean)):  # every weight of the column 448, or zero
        w2 = c["w2"].view(torch.uint8).clone().view(9, h // 16, i // 32, 2, 16, 16)
        w2[:, col // 16, :, :, col % 16] = code
        to["w2"] = w2.view(9, h, i)
    got, want = prompt.experts(**c), prompt.experts(**dict(c, **clean))
    keep = [n for n in range(h) if n != col]
    assert not bool(got[:, col].isfinite().all()) and bool(want.isfinite().all())
    assert float(want.float().abs().max()) > 2.0**110
    assert torch.equal(got[:, keep], want[:, keep])


def test_experts_of_the_most_elements(gpu_device):
    """As many elements as a call takes: rows past the rounding that is launched beside the
    sort (262144 of them) against 64 bits."""
    t, h, at = (1 << 19) - 1, 1 << 16, [0, 262143, 262144, 262145, 524286]
    c = dict(_experts_case(gpu_device, len(at), h, 128, 2, 1, shared=False), residual=None)
    torch.cuda.empty_cache()
    x = torch.empty(t, h, dtype=torch.bfloat16, device=gpu_device)  # (what lies in the other rows is theirs)
    ids, wts = torch.ones(t, 1, dtype=torch.int32, device=gpu_device), torch.ones(t, 1, device=gpu_device)
    x[at], ids[at], wts[at] = c["x"], c["ids"], c["weights"]
    got = prompt.experts(**dict(c, x=x, ids=ids, weights=wts, out=x))[at]
    del x
    torch.cuda.empty_cache()
    _check_experts(dict(c, residual=torch.zeros_like(c["x"])), got)


@pytest.mark.parametrize("h,i,e,k", [(256, 128, 8, 2), (1152, 384, 3, 2), (512, 640, 4, 3), (2432, 512, 6, 1)])
def test_experts_batch_invariant(gpu_device, h, i, e, k):
    """A token's output has the same bits alone, in the smallest and the widest company, and in
    another place of the call; and it is right."""
    c = dict(_experts_case(gpu_device, 600, h, i, e, k), batch_invariant=True)
    c["ids"][5] = -1
    rows = ("x", "ids", "weights", "residual")
    want = prompt.experts(**c)
    _check_experts({n: v for n, v in c.items() if n != "batch_invariant"}, want)
    order = torch.randperm(600, generator=torch.Generator().manual_seed(h)).to(gpu_device)
    assert torch.equal(prompt.experts(**dict(c, **{n: c[n][order] for n in rows})), want[order])
    for first, n in [(0, 1), (7, 16), (3, 17), (100, 64), (100, 65), (90, 97), (1, 300)]:
        part = {r: c[r][first:first + n].contiguous() for r in rows}
        assert torch.equal(prompt.experts(**dict(c, **part)), want[first:first + n]), (first, n)
        if n <= 96:  # calls this small sum so in any case
            assert torch.equal(prompt.experts(**dict(c, batch_invariant=False, **part)), want[first:first + n])


def test_experts_of_no_tokens(gpu_device):
    c = _experts_case(gpu_device, 4, 256, 128, 8, 2)
    for k in ("x", "ids", "weights", "residual"):
        c[k] = c[k][:0]
    assert prompt.experts(**c).shape == (0, 256)


# ------------------------------------------------ each way to run, as callers may
WAYS = [(3, 272, 1024), (24, 272, 1024), (24, 64, 7168), (90, 2112, 256), (300, 528, 4096), (2050, 4112, 256)]


@pytest.mark.parametrize("m,n,k", WAYS)
def test_product_f32_strided_out(gpu_device, m, n, k):
    w, s = _matrix(n, k, gpu_device, 61)
    x = workloads.rows_bf16(m, k, gpu_device, seed=62)
    buf = torch.full((m + 2, n + 24), 3.0, device=gpu_device)
    got = prompt.product(x, w, s, out=buf[1:-1, 8:-16])
    assert torch.equal(got, prompt.product(x, w, s, dtype=torch.float32))
    assert bool((buf[0] == 3).all()) and bool((buf[-1] == 3).all())
    assert bool((buf[:, :8] == 3).all()) and bool((buf[:, -16:] == 3).all())


@pytest.mark.parametrize("m,n,k", [(1, 16, 65536), (30, 32, 65536), (100, 16, 65536), (4200, 16, 65536), (1, 65536, 128),
                                   (20, 65536, 128), (200, 65536, 256)])
def test_product_widest(gpu_device, m, n, k):
    """The largest K and N that a call takes, each way to run."""
    w, s = _matrix(n, k, gpu_device, 63)
    x = workloads.rows_bf16(m, k, gpu_device, seed=64)
    at = torch.tensor(sorted({0, m // 2, m - 1}))
    want, mag = ref.product(x[at].cpu(), w.cpu(), s.cpu())
    for dtype in (torch.bfloat16, torch.float32):
        _same(prompt.product(x, w, s, dtype=dtype)[at], want, mag, dtype == torch.float32, k)


@pytest.mark.parametrize("t,h,i", [(3, 256, 32768), (120, 128, 32768), (5, 65536, 128), (120, 65536, 128)])
def test_experts_widest(gpu_device, t, h, i):
    c = _experts_case(gpu_device, t, h, i, 1, 1)
    _check_experts(c, prompt.experts(**c))


def test_graph_replays_of_each_way_to_run(gpu_device):
    """Every way to run in one graph, replayed on new inputs with eager work between."""
    dev = gpu_device
    mats = [(_matrix(n, k, dev, 65), workloads.rows_bf16(m, k, dev, seed=66)) for m, n, k in WAYS]
    moe = [_experts_case(dev, t, 256, i, 8, 4) for t, i in ((9, 128), (90, 640), (200, 128), (200, 640))]

    def calls():
        out = [prompt.product(x, *w, dtype=d) for w, x in mats for d in (torch.bfloat16, torch.float32)]
        return out + [prompt.experts(**c, batch_invariant=b) for c in moe for b in (False, True)]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = calls()
    for step in range(4):
        for _, x in mats:
            x.copy_(workloads.rows_bf16(*x.shape, dev, seed=67 + step))
        for c in moe:
            c["x"].copy_(workloads.rows_bf16(*c["x"].shape, dev, seed=77 + step))
            c["ids"].copy_(torch.randint(-1, 8, c["ids"].shape, device=dev).int())
        graph.replay()
        got = [o.clone() for o in outs]
        want = calls()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------- streams, graphs, repeats
def test_repeats_and_streams(gpu_device):
    """The same bits from call to call, and from two streams at once."""
    c = _experts_case(gpu_device, 200, 512, 256, 16, 4)
    w, s = _matrix(528, 512, gpu_device, 9)
    want, wantp = prompt.experts(**c), prompt.product(c["x"], w, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu_device) for _ in range(2)]
    got = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                got.append((prompt.experts(**c), prompt.product(c["x"], w, s)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) and torch.equal(b, wantp) for a, b in got)


def test_graph_replays(gpu_device):
    """Captured calls replayed on new inputs with eager work between, two graphs in turn."""
    c = _experts_case(gpu_device, 70, 256, 128, 8, 2)
    a = _append_case(gpu_device, [(0, 70)], False, False)
    w, s = _matrix(144, 256, gpu_device, 13)
    graphs = []
    for _ in range(2):
        prompt.experts(**c), prompt.product(c["x"], w, s), prompt.append(**a)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = prompt.experts(**c), prompt.product(c["x"], w, s)
            prompt.append(**a)
        graphs.append((gr, outs))
    for step in range(4):
        c["x"].copy_(workloads.rows_bf16(70, 256, gpu_device, seed=90 + step))
        c["ids"].copy_(torch.randint(-1, 8, (70, 2), device=gpu_device).int())
        a["kv_a"].copy_(torch.randn(70, 576, device=gpu_device))
        for gr, outs in graphs:
            a["caches"].kv.zero_()
            gr.replay()
            kv = a["caches"].kv.clone()
            want = prompt.experts(**c), prompt.product(c["x"], w, s)
            a["caches"].kv.zero_()
            prompt.append(**a)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(kv, a["caches"].kv)


# ------------------------------------------------------------- used together
def test_prompt_then_decode_attention(gpu_device):
    """Two prompts' normed rows through the projections' own weights into the caches, which
    the decode attention then reads: its selection and output against the oracle on the
    same caches."""
    dev, lens, ctx = gpu_device, [2300, 77], 4096
    w = workloads.proj_weights(dev, seed=31)
    step, caches = workloads.attn_case(lens, dev, seed=32, max_ctx=ctx)
    caches.kv.zero_(), caches.ikv.zero_(), caches.iks.zero_(), caches.kv_scale.zero_()
    cos, sin = workloads.rope_tables(ctx, dev)
    req = torch.cat([torch.full((n,), r, device=dev) for r, n in enumerate(lens)]).int()
    pos = torch.cat([torch.arange(n, device=dev) for n in lens]).int()
    x = workloads.rows_bf16(sum(lens), 7168, dev, seed=33)
    qkv = prompt.product(x, w.w_qkv, w.s_qkv)
    ik = prompt.product(x, w.w_ik, w.s_ik)
    assert qkv.shape == (sum(lens), N_QKV)
    prompt.append(qkv[:, Q_LORA:], ik, req, pos, step.page_table, caches, w.g_kv, w.g_ik, w.b_ik, cos, sin)
    rt = AttnRuntime(2, ctx, device=dev)
    out, dbg = rt.forward(step, caches, debug=True)
    torch.cuda.synchronize()
    rt.check_errors()
    rt.close()
    seq, pt, sel = step.seq_lens.cpu(), step.page_table.cpu(), dbg["topk"].cpu()
    assert torch.equal(sel, oatt.select_topk(dbg["scores"].cpu(), seq, pt))
    want = oatt.sparse_mla(step.q.cpu(), caches.kv.cpu(), caches.kv_scale.cpu(), sel)
    err = (out.cpu().float() - want.float()).abs()
    assert bool((err <= 2e-2 + 1e-2 * want.float().abs()).all()), float(err.max())  # the attention's own bounds
    # the rows are the projections': dequantised latents against the norm of the f64 products
    for r, n in enumerate(lens):
        t = torch.tensor([0, n // 2, n - 1])
        slots = pt[r, t // 64].long() * 64 + t % 64
        row = caches.kv.cpu()[slots].view(torch.float8_e4m3fn).double() * caches.kv_scale.cpu()[slots].double()[:, None]
        at = t + sum(lens[:r])
        y, _ = ref.product(x[at.to(dev)].cpu(), w.w_qkv.cpu(), w.s_qkv.cpu())
        lat = y[:, Q_LORA:Q_LORA + KV_LORA]
        lat = lat / (lat.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.g_kv.cpu().double()
        # product and latent in bf16 (2^-8 each), E4M3 (2^-4), a subnormal's half step 2^-10 of a scale
        # (<= 2^-7 of the largest)
        tol = (2.0**-8 + 2.0**-8 + 2.0**-4 + 2.0**-9) * lat.abs() + 2.0**-16 * row.abs().amax(-1, keepdim=True)
        assert bool(((row[:, :KV_LORA] - lat).abs() <= tol + 2.0**-7 * lat.square().mean().sqrt()).all())
        assert row.shape[1] == KV_LORA + PE_DIM


@pytest.mark.parametrize("raw", [False, True], ids=["scaled", "raw"])
def test_keys_beside_the_front_s(gpu_device, raw):
    """The cache rows of 16 tokens by the front launch, by the append on the projections that
    the front computes (bf16 rows times the weights), and by product and append, whose rows
    are rounded to E4M3 before the product: the first two are the same but for codes that
    hang on f32's last bits (the front's own test allows 2 % of the codes a step, 5 % of the
    few FP4 bytes), the third is off by that rounding."""
    dev, ctx = gpu_device, [1500, 70, 4097, 64, 2048, 2049, 300, 1, 65, 128, 129, 999, 5000, 63, 2, 4096]
    n = len(ctx)
    w = workloads.proj_weights(dev, seed=51)
    step, front = workloads.attn_case(ctx, dev, seed=52, max_ctx=8192)
    if raw:
        front.kv_scale = None
    mine, theirs = [AttnCaches(*(None if t is None else t.clone() for t in (front.ikv, front.iks, front.kv, front.kv_scale)))
                    for _ in range(2)]
    cos, sin = workloads.rope_tables(8192, dev)
    h = workloads.rows_bf16(n, 7168, dev, seed=53)
    rt = ProjRuntime(16, dev)
    rt.front(h, step.seq_lens, step.page_table, front, w, cos, sin)
    torch.cuda.synchronize()
    rt.check_errors()
    rt.close()
    req, pos = torch.arange(n, device=dev).int(), step.seq_lens - 1
    x = olayer.rmsnorm(h.cpu(), w.g_in.cpu()).to(torch.bfloat16)
    exact = [(x.double() @ ref.weight(m.cpu(), s.cpu()).T).float().to(dev) for m, s in ((w.w_qkv, w.s_qkv), (w.w_ik, w.s_ik))]
    rounded = [prompt.product(x.to(dev), m, s, dtype=torch.float32) for m, s in ((w.w_qkv, w.s_qkv), (w.w_ik, w.s_ik))]
    for (qkv, ik), caches in ((exact, theirs), (rounded, mine)):
        prompt.append(qkv[:, Q_LORA:], ik, req, pos, step.page_table, caches, w.g_kv, w.g_ik, w.b_ik, cos, sin)
    slot = olayer.slot_of(step.page_table.cpu(), pos.cpu())
    page, t = slot // 64, slot % 64

    def rows(c):
        scale = torch.ones(n) if raw else c.kv_scale.cpu()[slot]
        return codecs.e4m3_decode(c.kv.cpu()[slot]).double() * scale.double()[:, None], scale.double()[:, None]

    (a, s), (b, _), (c, _) = rows(front), rows(theirs), rows(mine)
    assert float((a != b).double().mean()) <= 0.02
    assert bool(((a - b).abs() <= torch.maximum(a.abs(), b.abs()) * 2.0**-3 + s * 2.0**-9).all())
    for name in ("ikv", "iks"):
        p, q = (getattr(k, name).cpu() for k in (front, theirs))
        at = (page, slice(None), t) if name == "ikv" else (page, slice(None), t % 16 * 4 + t // 16)
        assert float((p[at] != q[at]).double().mean()) <= 0.05, name
        q[at] = p[at]
        assert torch.equal(p, q), name  # every other place is as it was
    # rows in E4M3 are 2^-4 off at most, each by itself: 2^-4 of the sums' norm; each side's own codes 2^-4
    rel = (c - a).norm(dim=1) / a.norm(dim=1)
    print("rows off by", [round(float(r), 4) for r in rel], flush=True)
    assert bool((rel <= 3 * 2.0**-4).all())
    assert float((rounded[0] - exact[0]).norm() / exact[0].norm()) <= 2.0**-4


def test_experts_against_the_decode_launch(gpu_device):
    """A decode step's MoE and the prompt's experts on its own routing: the same products
    (the launch rounds its f32 normed rows to FP8, the prompt's rows come in bf16)."""
    dev = gpu_device
    w = workloads.fp8_moe_weights(FP8_MOE, dev, seed=41)
    a = workloads.rows_bf16(8, FP8_MOE.hidden, dev, seed=42)
    rt = MoeRuntime(FP8_MOE, 8, device=dev)
    want, dbg = rt.forward_fp8(a, w, debug=True)
    torch.cuda.synchronize()
    rt.check_errors()
    rt.close()
    x = a.float() * torch.rsqrt(a.float().square().mean(-1, keepdim=True) + FP8_MOE.eps) * w.g_post.float()
    got = prompt.experts(x.to(torch.bfloat16), dbg["topk_ids"], dbg["topk_w"], w.w13, w.s13, w.w2, w.s2, residual=a)
    # a bf16 row is 2^-8 off: at most 2^-8 / 2^-4 of the codes a step (2^-3) over, 2^-3 sqrt(2^-4) = 0.031 of
    # each product at the very worst (all of them at a border); the sums' sizes are the launch's own
    y = dbg["y"].double()
    d = (got.double() - want.double())
    assert float(d.norm()) <= 2 * 0.031 * float(y.norm()) + 2.0**-7 * float(want.double().norm())
    assert bool((d.abs() <= 6 * 2 * 0.031 * y.square().mean().sqrt() + 2.0**-7 * want.double().abs()).all())


def test_experts_on_the_decode_launch_s_rows(gpu_device):
    """As above, on rows that both sides round to the same codes: in every 8 columns one of
    size 2, three of size 1 and four of 1/2, whose mean square is 1, so that the launch's norm
    leaves them (5e-7 off, which a code of 448 / 2^j does not hang on), and with experts whose
    sum outweighs the residual. What is left is the module's head's: mids over a border, and
    the outputs' rounding."""
    dev = gpu_device
    w = workloads.fp8_moe_weights(FP8_MOE, dev, seed=43)
    w.g_post.fill_(1.0)
    w.s2 *= 4096.0
    g = torch.Generator(device=dev).manual_seed(44)
    size = torch.tensor([2.0, 1.0, 1.0, 1.0, 0.5, 0.5, 0.5, 0.5], device=dev)
    order = torch.rand(8, FP8_MOE.hidden // 8, 8, generator=g, device=dev).argsort(-1)
    sign = torch.randint(0, 2, (8, FP8_MOE.hidden), generator=g, device=dev) * 2 - 1
    a = (size[order].view(8, -1) * sign).to(torch.bfloat16)
    rt = MoeRuntime(FP8_MOE, 8, device=dev)
    want, dbg = rt.forward_fp8(a, w, debug=True)
    torch.cuda.synchronize()
    rt.check_errors()
    rt.close()
    got = prompt.experts(a, dbg["topk_ids"], dbg["topk_w"], w.w13, w.s13, w.w2, w.s2, residual=a)
    d, y = got.double() - want.double(), dbg["y"].double()
    print(f"{float(d.norm() / want.double().norm()):.2e}", flush=True)
    assert float(y.norm()) > 4 * float(a.double().norm())
    assert float(d.norm()) <= 0.0056 * float(y.norm()) + 2.0**-8 * float(want.double().norm())
