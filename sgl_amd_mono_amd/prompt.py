"""The layer's work at prompt widths: up to 1048576 rows a call on the layer's own weights
and caches, where the decode launches take a step of a few.

* ``product``: rows, rounded to E4M3, times one FP8 matrix with a scale for each 128 x 128
  block: the projections' weights as they are. (``layer.ProjRuntime`` multiplies a decode
  step's rows in bf16, unrounded: a projection of ``product`` is 2.6 % of its norm off that.)
* ``append``: a prompt's keys into the MLA cache and the index plane (what the front
  launch writes for a decode step's rows, from the same projections)
* ``experts``: the routed and the shared FP8 experts (the products of
  ``moe.MoeRuntime.forward_fp8``, behind a router of the caller's)
* ``index_query``, ``page_scores``, ``select_pages``, ``attention``: a prompt's own sparse
  attention. Where a decode step's row selects its 2048 best keys one at a time, a prompt's
  token selects pages of 64 keys by the best index score in each, and attends to their keys:
  beyond 2048 keys not those of the layer's definition.
* ``tree_attention``: attention of a tree of drafted tokens to its request's keys and to
  those of the draft that each token's mask lets it see

The functions keep no state. They check the tensors, take their scratch from torch's
allocator and enqueue on the current stream of the tensors' device, so calls on several
streams do not disturb each other, and a call may be captured in a graph. Operands made
on another stream are the caller's to order, as for any torch operator.

A call takes at most 1048576 rows (``experts``: tokens times (picks + 1), 116508 tokens at
8 picks) and 2^35 elements of them. Scratch: a product K * (1 + 1/32) bytes a row, and f32
parts where its tiles are few; ``experts`` mostly 2 * H bytes for each token's every pick
(1.2 GB for 8192 tokens of 7168 with 8 picks and the shared expert), so a long prompt goes
through it in pieces of some thousand tokens; both attentions f32 parts, for up to 256 tokens
or 1024 nodes of 32 heads at most 512 or 1024 of [heads, 512] (34 or 67 MB). A captured graph
keeps its calls' scratch.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .attn import PAGE, SOFTMAX_SCALE, TOPK, AttnCaches
from .layer import INDEX_DIM, INDEX_HEADS, KV_LORA, PE_DIM
from .moe import FP8_TYPES
from .runtime import need as _need

MAX_COLUMNS = 8192  # pages that a call scores, selects from or lists for a token: 524288 keys


# The current stream's handle without a Stream object around it, which takes longer to make
# than a short launch takes to enqueue.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def need(t: torch.Tensor, name: str, shape: tuple, dtypes, dev: torch.device) -> None:
    """runtime.need, which names what is wrong, behind a quick look that finds nothing wrong:
    a short call checks eleven tensors and takes no longer than its launch."""
    try:
        if (t.dtype is dtypes or t.dtype in dtypes) and t.shape == shape and t.get_device() == dev.index and t.is_contiguous():
            return
    except (AttributeError, TypeError):
        pass
    _need(t, name, shape, dtypes, dev)


def _gpu(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a tensor on a GPU, got {t.device}")
    return t.device


def _rows(t: torch.Tensor, name: str, shape: tuple, dtype, dev: torch.device) -> int:
    """Raise ValueError unless ``t`` is [rows, columns] of this shape, dtype and device whose
    columns lie together; returns the elements from a row to the next (the columns, where
    there is no next)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a tensor, got {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name}: expected device {dev}, got {t.device}")
    rows, columns = shape
    if rows <= 1:
        if rows and columns > 1 and t.stride(1) != 1:
            raise ValueError(f"{name}: expected columns that lie together (strides {t.stride()})")
        return -(-columns // 8) * 8
    stride = t.stride()
    if (stride[1] != 1 and columns > 1) or stride[0] < columns:
        raise ValueError(f"{name}: expected columns that lie together and rows apart (strides {stride})")
    return stride[0]


def _apart(a: torch.Tensor, a_stride: int, b: torch.Tensor, b_stride: int) -> bool:
    """Whether two matrices of bytes-apart rows share no element: neither's memory reaches the
    other's, or both are columns of one wider matrix, side by side."""
    if not a.numel() or not b.numel():
        return True
    sa, sb = a_stride * a.element_size(), b_stride * b.element_size()
    wa, wb = a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + (a.shape[0] - 1) * sa + wa <= pb or pb + (b.shape[0] - 1) * sb + wb <= pa:
        return True
    return sa == sb and (pb - pa) % sa >= wa and (pb - pa) % sa + wb <= sa


def _enqueue(dev: torch.device, fn, args) -> None:
    if torch.cuda.current_device() == dev.index:
        rc = fn(C.byref(args), _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(C.byref(args), _raw_stream(dev.index))
    if rc:
        _lib.check(rc)


def _workspace(args, nbytes: int, dev: torch.device) -> torch.Tensor | None:
    if nbytes < 0:
        raise ValueError(_lib.lib().mono_last_error().decode(errors="replace"))
    if nbytes == 0:
        return None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def product(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, out: torch.Tensor | None = None,
            dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x`` [rows, K] bf16 (rows may lie apart, each 16-byte aligned) times ``w`` [N, K]
    E4M3 in the (16, 16) layout with scales ``s`` f32 [ceil(N / 128), K / 128] -> [rows, N]
    in ``dtype`` (bf16 or f32; ``out``'s own where that is given). The rows are rounded to
    E4M3 with a scale for each 128 columns, whatever ``dtype`` (the decode launches round
    none of a projection's); a row that holds a NaN or an infinity has NaN
    outputs. N % 16 == 0, K % 128 == 0. ``out`` must share no memory with ``x``."""
    dev = _gpu(x, "x")
    if x.dim() != 2 or not isinstance(w, torch.Tensor) or w.dim() != 2:
        raise ValueError(f"x and w: expected [rows, K] and [N, K], got {tuple(x.shape)} and {tuple(getattr(w, 'shape', ()))}")
    (m, k), n = x.shape, w.shape[0]
    stride = _rows(x, "x", (m, k), torch.bfloat16, dev)
    need(w, "w", (n, k), FP8_TYPES, dev)
    need(s, "s", (-(-n // 128), k // 128), torch.float32, dev)
    if out is not None:
        if not isinstance(out, torch.Tensor):
            raise ValueError(f"out: expected a tensor, got {type(out).__name__}")
        dtype = out.dtype
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"out: expected dtype torch.bfloat16 or torch.float32, got {dtype}")
    if out is None:
        out = torch.empty(m, n, dtype=dtype, device=dev)
        out_stride = n
    else:
        out_stride = _rows(out, "out", (m, n), dtype, dev)
        if not _apart(x, stride, out, out_stride):
            raise ValueError("out: shares memory with x")
    args = _lib.PromptProductArgs(x=x.data_ptr(), x_stride=stride, w=w.data_ptr(), s=s.data_ptr(), out=out.data_ptr(),
                                  out_stride=out_stride, out_f32=dtype == torch.float32, rows=m, n=n, k=k)
    lib = _lib.lib()
    ws = _workspace(args, lib.mono_prompt_product_workspace(m, n, k), dev)  # noqa: F841 (held over the call)
    _enqueue(dev, lib.mono_prompt_product, args)
    return out


def append(kv_a: torch.Tensor, ik: torch.Tensor, req: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor,
           caches: AttnCaches, g_kv: torch.Tensor, g_ik: torch.Tensor, b_ik: torch.Tensor, rope_cos: torch.Tensor,
           rope_sin: torch.Tensor, slot_pos: torch.Tensor | None = None) -> None:
    """Write the keys of ``tokens`` tokens into ``caches`` in place, as the front launch
    writes a decode step's: ``kv_a`` [tokens, 576] (latent 512 | k_pe 64) and ``ik``
    [tokens, 128], bf16 or f32 (both alike; rows may lie apart), are the projections before
    their norms and rotation. Token i is position ``pos[i]`` of request ``req[i]``, a row
    of ``page_table`` [requests, pages] (all i32). A token whose request, position (below
    the rows of ``rope_cos`` / ``rope_sin`` and what the page table covers) or page is out
    of range is a pad and writes nothing; two tokens must not share a slot.

    With ``slot_pos`` (i32 [tokens]) token i's key is rotated for ``pos[i]`` and written to the
    slot of position ``slot_pos[i]``: the tokens of a drafted tree may share a position, but
    each has a slot of its own (``tree_attention``)."""
    dev = _gpu(kv_a, "kv_a")
    if kv_a.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"kv_a: expected dtype torch.bfloat16 or torch.float32, got {kv_a.dtype}")
    t = kv_a.shape[0] if kv_a.dim() == 2 else -1
    kv_stride = _rows(kv_a, "kv_a", (t, KV_LORA + PE_DIM), kv_a.dtype, dev)
    ik_stride = _rows(ik, "ik", (t, INDEX_DIM), kv_a.dtype, dev)
    need(req, "req", (t,), torch.int32, dev)
    need(pos, "pos", (t,), torch.int32, dev)
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise ValueError(f"page_table: expected [requests, pages], got {tuple(getattr(page_table, 'shape', ()))}")
    need(page_table, "page_table", tuple(page_table.shape), torch.int32, dev)
    if not isinstance(caches.ikv, torch.Tensor) or caches.ikv.dim() != 4:
        raise ValueError(f"ikv: expected [pages, 4, {PAGE}, 16], got {tuple(getattr(caches.ikv, 'shape', ()))}")
    pages = caches.ikv.shape[0]
    need(caches.ikv, "ikv", (pages, 4, PAGE, 16), torch.uint8, dev)
    need(caches.iks, "iks", (pages, 4, PAGE), torch.uint8, dev)
    need(caches.kv, "kv", (pages * PAGE, KV_LORA + PE_DIM), FP8_TYPES, dev)
    if caches.kv_scale is not None:  # None: raw E4M3 rows (scale 1)
        need(caches.kv_scale, "kv_scale", (pages * PAGE,), torch.float32, dev)
    need(g_kv, "g_kv", (KV_LORA,), torch.bfloat16, dev)
    need(g_ik, "g_ik", (INDEX_DIM,), torch.float32, dev)
    need(b_ik, "b_ik", (INDEX_DIM,), torch.float32, dev)
    if not isinstance(rope_cos, torch.Tensor) or rope_cos.dim() != 2 or rope_cos.shape[1] != PE_DIM // 2:
        raise ValueError(f"rope_cos: expected [max_pos, {PE_DIM // 2}], got {tuple(getattr(rope_cos, 'shape', ()))}")
    need(rope_cos, "rope_cos", tuple(rope_cos.shape), torch.float32, dev)
    need(rope_sin, "rope_sin", tuple(rope_cos.shape), torch.float32, dev)
    args = _lib.PromptAppendArgs(
        kv_a=kv_a.data_ptr(), kv_stride=kv_stride, ik=ik.data_ptr(), ik_stride=ik_stride, f32=kv_a.dtype == torch.float32,
        tokens=t, req=req.data_ptr(), pos=pos.data_ptr(), page_table=page_table.data_ptr(), requests=page_table.shape[0],
        pt_stride=page_table.shape[1], n_pages=pages, max_pos=rope_cos.shape[0], g_kv=g_kv.data_ptr(),
        g_ik=g_ik.data_ptr(), b_ik=b_ik.data_ptr(), rope_cos=rope_cos.data_ptr(), rope_sin=rope_sin.data_ptr(),
        kv=caches.kv.data_ptr(), kv_scale=_lib.ptr(caches.kv_scale), ikv=caches.ikv.data_ptr(), iks=caches.iks.data_ptr(),
    )  # fmt: skip
    if slot_pos is None:
        _enqueue(dev, _lib.lib().mono_prompt_append, args)
    else:
        need(slot_pos, "slot_pos", (t,), torch.int32, dev)
        at = slot_pos.data_ptr()
        _enqueue(dev, lambda a, stream: _lib.lib().mono_prompt_append_at(a, at, stream), args)


def experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, w13: torch.Tensor, s13: torch.Tensor,
            w2: torch.Tensor, s2: torch.Tensor, residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
            shared: bool = True, batch_invariant: bool = False) -> torch.Tensor:
    """``residual[t] + shared(x[t]) + sum_j weights[t, j] * expert_ids[t, j](x[t])``, bf16
    [tokens, H]. ``x`` [tokens, H] bf16 are the normed rows, ``ids`` i32 and ``weights``
    f32 [tokens, picks] the router's answer (an id outside the routed experts is routed
    nowhere), the weights and scales those of ``moe.Fp8MoeWeights``. With ``shared`` the
    last expert is the shared one (every token, weight 1) and ids name the others. Rows of
    ``x``, ``residual`` and ``out`` may lie apart; ``out`` may be ``residual`` or ``x`` itself.

    Wide calls (above 96 tokens with more than 11 picks a routed expert on average) sum their
    up products on the FP8 MFMA, 1.4e-5 off for each 128 of them, narrower ones exactly but
    for f32's rounding. With ``batch_invariant`` every call does as the narrower ones do: a
    token's output then has the same bits whatever other tokens are in the call."""
    dev = _gpu(x, "x")
    if x.dim() != 2 or not isinstance(ids, torch.Tensor) or ids.dim() != 2:
        raise ValueError(f"x and ids: expected [tokens, H] and [tokens, picks], got {tuple(x.shape)} and "
                         f"{tuple(getattr(ids, 'shape', ()))}")  # fmt: skip
    if not isinstance(w13, torch.Tensor) or w13.dim() != 3 or w13.shape[0] <= bool(shared) or w13.shape[1] % 256:
        raise ValueError(f"w13: expected [experts, 2 I, H] with I a multiple of 128, got {tuple(getattr(w13, 'shape', ()))}")
    (t, h), k, e, i = x.shape, ids.shape[1], w13.shape[0], w13.shape[1] // 2
    x_stride = _rows(x, "x", (t, h), torch.bfloat16, dev)
    need(ids, "ids", (t, k), torch.int32, dev)
    need(weights, "weights", (t, k), torch.float32, dev)
    need(w13, "w13", (e, 2 * i, h), FP8_TYPES, dev)
    need(s13, "s13", (e, 2 * i // 128, h // 128), torch.float32, dev)
    need(w2, "w2", (e, h, i), FP8_TYPES, dev)
    need(s2, "s2", (e, h // 128, i // 128), torch.float32, dev)
    res_stride = h if residual is None else _rows(residual, "residual", (t, h), torch.bfloat16, dev)
    if out is None:
        out, out_stride = torch.empty(t, h, dtype=torch.bfloat16, device=dev), h
    else:
        out_stride = _rows(out, "out", (t, h), torch.bfloat16, dev)
        same = residual is None or (out.data_ptr() == residual.data_ptr() and out_stride == res_stride)
        if not same and not _apart(residual, res_stride, out, out_stride):
            raise ValueError("out: shares memory with residual, and is not residual itself")
    args = _lib.PromptExpertsArgs(
        x=x.data_ptr(), x_stride=x_stride, ids=ids.data_ptr(), weights=weights.data_ptr(), w13=w13.data_ptr(),
        s13=s13.data_ptr(), w2=w2.data_ptr(), s2=s2.data_ptr(), residual=_lib.ptr(residual), residual_stride=res_stride,
        out=out.data_ptr(), out_stride=out_stride, tokens=t, picks=k, experts=e - bool(shared), shared=bool(shared),
        hidden=h, inter=i, batch_invariant=bool(batch_invariant),
    )  # fmt: skip
    lib = _lib.lib()
    ws = _workspace(args, lib.mono_prompt_experts_workspace(C.byref(args)), dev)  # noqa: F841 (held over the call)
    _enqueue(dev, lib.mono_prompt_experts, args)
    return out


def index_query(x: torch.Tensor, pos: torch.Tensor, rope_cos: torch.Tensor,
                rope_sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The FP4 index queries of tokens at ``pos`` (i32 [tokens]): ``x`` [tokens, 64 * 128] bf16
    or f32 (rows may lie apart, each 16-byte aligned) is the projection before its rotation.
    Returns ``(iq, iqs)``, u8 [tokens, 64, 64] and [tokens, 64, 4], as ``attn.AttnStep`` and
    ``page_scores`` take them. A token whose position has no row in ``rope_cos`` / ``rope_sin`` is
    a pad: zeros."""
    dev = _gpu(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"x: expected dtype torch.bfloat16 or torch.float32, got {x.dtype}")
    t = x.shape[0] if x.dim() == 2 else -1
    stride = _rows(x, "x", (t, INDEX_HEADS * INDEX_DIM), x.dtype, dev)
    need(pos, "pos", (t,), torch.int32, dev)
    if not isinstance(rope_cos, torch.Tensor) or rope_cos.dim() != 2 or rope_cos.shape[1] != PE_DIM // 2:
        raise ValueError(f"rope_cos: expected [max_pos, {PE_DIM // 2}], got {tuple(getattr(rope_cos, 'shape', ()))}")
    need(rope_cos, "rope_cos", tuple(rope_cos.shape), torch.float32, dev)
    need(rope_sin, "rope_sin", tuple(rope_cos.shape), torch.float32, dev)
    iq = torch.empty(t, INDEX_HEADS, INDEX_DIM // 2, dtype=torch.uint8, device=dev)
    iqs = torch.empty(t, INDEX_HEADS, INDEX_DIM // 32, dtype=torch.uint8, device=dev)
    args = _lib.PromptQueryArgs(x=x.data_ptr(), x_stride=stride, f32=x.dtype == torch.float32, tokens=t, pos=pos.data_ptr(),
                                max_pos=rope_cos.shape[0], rope_cos=rope_cos.data_ptr(), rope_sin=rope_sin.data_ptr(),
                                iq=iq.data_ptr(), iqs=iqs.data_ptr())
    _enqueue(dev, _lib.lib().mono_prompt_query, args)
    return iq, iqs


def _tokens_of(req: torch.Tensor, pos: torch.Tensor, page_table: torch.Tensor, t: int, dev: torch.device) -> None:
    need(req, "req", (t,), torch.int32, dev)
    need(pos, "pos", (t,), torch.int32, dev)
    _table(page_table, dev)


def _pages_number(v: int, name: str) -> None:
    if not isinstance(v, int) or not 0 <= v <= MAX_COLUMNS:
        raise ValueError(f"{name}: expected a number of pages in [0, {MAX_COLUMNS}], got {v!r}")


def _table(page_table: torch.Tensor, dev: torch.device) -> None:
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise ValueError(f"page_table: expected [requests, pages], got {tuple(getattr(page_table, 'shape', ()))}")
    need(page_table, "page_table", tuple(page_table.shape), torch.int32, dev)


def page_scores(iq: torch.Tensor, iqs: torch.Tensor, iw: torch.Tensor, req: torch.Tensor, pos: torch.Tensor,
                page_table: torch.Tensor, caches: AttnCaches, columns: int | None = None) -> torch.Tensor:
    """The best index score in each page that a token sees: f32 [tokens, columns], for pages 0
    .. ``columns`` - 1 of its request (default: all that ``page_table`` [requests, pages] has;
    at most 8192). ``iq`` / ``iqs`` are the tokens' index queries (``index_query``), ``iw`` bf16
    [tokens, 64] their head weights; token i is position ``pos[i]`` of request ``req[i]`` (i32),
    and a key's score the decode launches' index score, summed in f32: off by 12 roundings at most,
    2^-24 each, of the sum of all heads' |weight x product| (where a query's and a key's scales lie
    within 2^7 of each other, so that f32 holds their products exactly). -infinity where the token sees no key
    of the page, NaN where the score of one is (a NaN product, which the decode launches take for 0)."""
    dev = _gpu(iq, "iq")
    t = iq.shape[0] if iq.dim() == 3 else -1
    need(iq, "iq", (t, INDEX_HEADS, INDEX_DIM // 2), torch.uint8, dev)
    need(iqs, "iqs", (t, INDEX_HEADS, INDEX_DIM // 32), torch.uint8, dev)
    need(iw, "iw", (t, INDEX_HEADS), torch.bfloat16, dev)
    _tokens_of(req, pos, page_table, t, dev)
    if not isinstance(caches.ikv, torch.Tensor) or caches.ikv.dim() != 4:
        raise ValueError(f"ikv: expected [pages, 4, {PAGE}, 16], got {tuple(getattr(caches.ikv, 'shape', ()))}")
    pages = caches.ikv.shape[0]
    need(caches.ikv, "ikv", (pages, 4, PAGE, 16), torch.uint8, dev)
    need(caches.iks, "iks", (pages, 4, PAGE), torch.uint8, dev)
    columns = page_table.shape[1] if columns is None else columns
    _pages_number(columns, "columns")
    out = torch.empty(t, columns, dtype=torch.float32, device=dev)
    args = _lib.PromptScoresArgs(
        iq=iq.data_ptr(), iqs=iqs.data_ptr(), iw=iw.data_ptr(), tokens=t, req=req.data_ptr(), pos=pos.data_ptr(),
        page_table=page_table.data_ptr(), requests=page_table.shape[0], pt_stride=page_table.shape[1], n_pages=pages,
        ikv=caches.ikv.data_ptr(), iks=caches.iks.data_ptr(), out=out.data_ptr(), columns=columns,
    )  # fmt: skip
    _enqueue(dev, _lib.lib().mono_prompt_scores, args)
    return out


def select_pages(scores: torch.Tensor, pos: torch.Tensor, picks: int = TOPK // PAGE, first: int = 0, last: int = 1) -> torch.Tensor:
    """The pages that each token reads, i32 [tokens, picks] ascending, -1 behind them: of the
    pages 0 .. ``pos[i]`` // 64 of ``scores`` f32 [tokens, columns] (rows may lie apart) the
    ``first`` first and the ``last`` last (the token's own page among them), and the best-scored
    others, exactly, the lowest page of equal ones first (+0 above -0, a NaN by its bits). A token that
    sees at most ``picks`` pages reads all of them (with the default 32, every key of up to
    2048, as a decode step's row does). ``pos[i]`` < 0 is a pad: all -1, and so are all rows of
    ``scores`` without columns."""
    dev = _gpu(scores, "scores")
    if scores.dim() != 2:
        raise ValueError(f"scores: expected [tokens, columns], got {tuple(scores.shape)}")
    for name, v in (("picks", picks), ("first", first), ("last", last)):
        _pages_number(v, name)
    t, columns = scores.shape
    stride = max(_rows(scores, "scores", (t, columns), torch.float32, dev), columns)
    need(pos, "pos", (t,), torch.int32, dev)
    pages = torch.empty(t, picks, dtype=torch.int32, device=dev)
    if columns == 0:  # of no pages none is picked (a call of no tokens looks at the numbers all the same)
        pages.fill_(-1)
        t = 0
    args = _lib.PromptSelectArgs(scores=scores.data_ptr(), stride=stride, tokens=t, columns=columns or 1, pos=pos.data_ptr(),
                                 picks=picks, first=first, last=last, pages=pages.data_ptr())
    _enqueue(dev, _lib.lib().mono_prompt_select, args)
    return pages


def _latents(q: torch.Tensor, caches: AttnCaches, out: torch.Tensor | None, dev: torch.device) -> tuple[int, torch.Tensor]:
    """The checks that both attentions share: the cache's pages and ``out``."""
    if q.dim() != 3 or q.shape[2] != KV_LORA + PE_DIM:
        raise ValueError(f"q: expected [tokens, heads, {KV_LORA + PE_DIM}], got {tuple(q.shape)}")
    t, heads = q.shape[:2]
    need(q, "q", (t, heads, KV_LORA + PE_DIM), torch.bfloat16, dev)
    kv = caches.kv
    if not isinstance(kv, torch.Tensor) or kv.dim() != 2 or kv.shape[0] % PAGE:
        raise ValueError(f"kv: expected [pages * {PAGE}, {KV_LORA + PE_DIM}], got {tuple(getattr(kv, 'shape', ()))}")
    slots = kv.shape[0]
    need(kv, "kv", (slots, KV_LORA + PE_DIM), FP8_TYPES, dev)
    if caches.kv_scale is not None:  # None: raw E4M3 rows (scale 1)
        need(caches.kv_scale, "kv_scale", (slots,), torch.float32, dev)
    if out is None:
        out = torch.empty(t, heads, KV_LORA, dtype=torch.bfloat16, device=dev)
    else:
        need(out, "out", (t, heads, KV_LORA), torch.bfloat16, dev)
        b = out.data_ptr()
        for name, v in (("q", q), ("kv", kv), ("kv_scale", caches.kv_scale)):
            a = 0 if v is None else v.data_ptr()
            if a and a < b + 2 * out.numel() and b < a + v.element_size() * v.numel():
                raise ValueError(f"out: shares memory with {name}")
    return slots // PAGE, out


def attention(q: torch.Tensor, req: torch.Tensor, pos: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor,
              caches: AttnCaches, softmax_scale: float = SOFTMAX_SCALE, out: torch.Tensor | None = None) -> torch.Tensor:
    """Sparse MLA attention of a prompt's tokens: ``q`` bf16 [tokens, heads, 576] (absorbed
    latent query 512 | rotated query 64; up to 128 heads) over the cached rows of the pages that
    each token lists in ``pages`` (i32 [tokens, picks]: ``select_pages``; numbers of pages of
    its request, -1: none), as far as their positions are at most the token's own. Returns
    [tokens, heads, 512] bf16, what the attention launch of a decode step hands on.

    Token i is position ``pos[i]`` of request ``req[i]``, a row of ``page_table`` [requests,
    pages] (all i32). A listed page outside the table or the pool is none, one that is listed
    twice counts twice. A token that sees no key has zeros. Keys that a token does not see may
    hold anything. ``out`` must share no memory with the other arguments (``q`` and the cache are
    looked at).

    An element of ``q`` is held to 2^-21.8 of its head's largest (2^-17.8 in the last 64 dims),
    which is all of bf16 for those above 2^-14 (2^-10) of it; a head of ``q`` that is not finite has
    NaN outputs. A logit is summed on the FP8 matrix instruction, off by up to 2^-16 of the sum of its
    terms' magnitudes (as measured); a probability is rounded to bf16 before the values' sum, which is f32.
    Outputs are 0.0017 to 0.0021 of their norm from 64 bits, of which bf16 alone makes 0.0017. The
    same call gives the same bits, but a token's bits are not its own in any company: how many
    tokens a call has decides whether a token's pages are summed in parts."""
    dev = _gpu(q, "q")
    n_pages, out = _latents(q, caches, out, dev)
    t, heads = q.shape[:2]
    _tokens_of(req, pos, page_table, t, dev)
    if not isinstance(pages, torch.Tensor) or pages.dim() != 2:
        raise ValueError(f"pages: expected [tokens, picks], got {tuple(getattr(pages, 'shape', ()))}")
    picks = pages.shape[1]
    need(pages, "pages", (t, picks), torch.int32, dev)
    args = _lib.PromptAttentionArgs(
        q=q.data_ptr(), tokens=t, heads=heads, req=req.data_ptr(), pos=pos.data_ptr(), pages=pages.data_ptr(), picks=picks,
        page_table=page_table.data_ptr(), requests=page_table.shape[0], pt_stride=page_table.shape[1], n_pages=n_pages,
        kv=caches.kv.data_ptr(), kv_scale=_lib.ptr(caches.kv_scale), softmax_scale=softmax_scale, out=out.data_ptr(),
    )  # fmt: skip
    lib = _lib.lib()
    ws = _workspace(args, lib.mono_prompt_attention_workspace(t, heads, picks), dev)  # noqa: F841 (held over the call)
    _enqueue(dev, lib.mono_prompt_attention, args)
    return out


def tree_attention(q: torch.Tensor, starts: torch.Tensor, prefix: torch.Tensor, mask: torch.Tensor, page_table: torch.Tensor,
                   caches: AttnCaches, softmax_scale: float = SOFTMAX_SCALE, out: torch.Tensor | None = None) -> torch.Tensor:
    """MLA attention of drafted tokens, a tree a request, over the whole cached prefix: ``q`` bf16
    [nodes, heads, 576] as ``attention`` takes it -> [nodes, heads, 512] bf16. Request r (a row
    of ``page_table``) has ``prefix[r]`` keys and the nodes ``starts[r]`` .. ``starts[r + 1]`` - 1
    (i32 [requests] and [requests + 1]); the key of its node i lies at position ``prefix[r]`` + i
    (``append`` with ``slot_pos``). A node sees the prefix and, for each bit j of its ``mask``
    (i64 [nodes]: the node itself and its ancestors), the key at ``prefix[r]`` + j. A node of no
    request, and one that sees nothing, has zeros. ``out`` must share no memory with the other
    arguments (``q`` and the cache are looked at). ``q``, logits and probabilities are held as in
    ``attention``; a node's bits hang on the call's other trees, which decide the parts that its
    pages are summed in, but not on how wide ``page_table`` is."""
    dev = _gpu(q, "q")
    n_pages, out = _latents(q, caches, out, dev)
    t, heads = q.shape[:2]
    _table(page_table, dev)
    requests, width = page_table.shape
    need(starts, "starts", (requests + 1,), torch.int32, dev)
    need(prefix, "prefix", (requests,), torch.int32, dev)
    need(mask, "mask", (t,), torch.int64, dev)
    args = _lib.PromptTreeArgs(
        q=q.data_ptr(), nodes=t, heads=heads, starts=starts.data_ptr(), prefix=prefix.data_ptr(), mask=mask.data_ptr(),
        page_table=page_table.data_ptr(), requests=requests, pt_stride=width, n_pages=n_pages, kv=caches.kv.data_ptr(),
        kv_scale=_lib.ptr(caches.kv_scale), softmax_scale=softmax_scale, out=out.data_ptr(),
    )  # fmt: skip
    lib = _lib.lib()
    ws = _workspace(args, lib.mono_prompt_tree_workspace(t, heads, width), dev)  # noqa: F841 (held over the call)
    _enqueue(dev, lib.mono_prompt_tree, args)
    return out
