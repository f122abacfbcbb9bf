"""Attention for a tree of drafted tokens over the paged ckv / kpe cache
(speculative decoding; destination-passing style).

    run(q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table, cu_drafts,
        tree_mask, sm_scale, output, lse) -> None

Request r has ``prefix_lens[r]`` cached tokens and the drafts
``cu_drafts[r] .. cu_drafts[r+1]-1`` (rows of ``q_nope`` / ``q_pe``), whose own
ckv / kpe rows are in the cache already, behind the prefix: the j-th draft at
position ``prefix_lens[r] + j`` of the request's ``block_table`` row.  A draft
sees the whole prefix and the drafts whose bits its row of ``tree_mask`` has
(``masks_from_parents`` makes the rows of a tree).  One draft per request with
its own bit set is plain dense decoding.

Unlike ``dsa_b200.attention.run``, which reads 2048 selected slots, this reads
every visible token.  The two are the same function where a draft sees at most
2048 tokens (the indexer then selects them all); beyond, a model that decodes
with the indexer's selection gets another distribution from dense rows, and a
chain of its drafts is verified by ``indexer.run_prefill`` and ``attention.run``.
``lse`` is the base-2 log-sum-exp of the scaled logits; a row that sees nothing
yields output 0 and lse -inf.

* Any 1 to 128 heads; up to ``64 * tree_mask.shape[1]`` drafts per request.
* ``ckv_cache`` ``[pages, 64, 512]`` and ``kpe_cache`` ``[pages, 64, 64]`` may be
  strided (pages and rows at multiples of 16 bytes), such as two slices of one
  ``[pages, 64, 576]`` cache; they are never copied.
* Cache rows that a mask hides may hold anything, infinities and NaN included.
  A visible row with NaN, or with an infinity that makes its logit +inf or NaN,
  makes the output NaN.  If the logit is -inf, whether an infinity among its values
  counts as 0 times infinity or as nothing is not defined.
* ``output`` may be ``q_nope`` itself; other outputs over an input are refused.
* Query rows outside of ``[cu_drafts[0], cu_drafts[-1])`` are left as they are.
* Lengths stay on the device; every launch goes to the current stream and can
  be captured into a CUDA graph (make one call on the capturing stream first,
  so that its workspace exists).  Calls that overlap need different streams;
  threads may call on one stream, whose calls then run one after the other.
  A graph uses the workspace of the stream that it was captured on: it must not
  run beside another one captured there, nor beside calls on that stream.
* Lengths that do not fit, page ids outside the pool and drafts that do not
  fit the mask set a sticky status bit (``device_status``), as for the other
  operators; with ``DSA_B200_CHECK=1`` each call synchronises and raises.
"""

from __future__ import annotations

import ctypes
import os

import torch

from . import _native, workspace

PAGE_SIZE = 64
DIM_CKV = 512
DIM_KPE = 64
MAX_HEADS = 128
MAX_MASK_WORDS = 64

_CHECK = os.environ.get("DSA_B200_CHECK", "0") not in ("", "0")
_ws_bytes: dict = {}  # device index -> dsa_tree_attention_workspace_bytes


def masks_from_parents(parents, words=None) -> list:
    """``tree_mask`` rows (lists of signed 64-bit words) of one request's drafts:
    ``parents[j]`` is the index of draft j's parent, below j, or -1 if it
    follows the prefix directly.  Every draft sees its ancestors and itself.
    Rows have as many words as the drafts need, or ``words``: a batch's trees
    need the largest one's."""
    bits = []
    for j, par in enumerate(parents):
        if not -1 <= par < j:
            raise ValueError(f"parents[{j}] is {par}: a parent comes before its children")
        bits.append((1 << j) | (bits[par] if par >= 0 else 0))
    need = max(1, (len(bits) + 63) // 64)
    if words is None:
        words = need
    elif words < need:
        raise ValueError(f"{len(bits)} drafts need {need} words, not {words}")
    rows = [[(m >> (64 * w)) & ((1 << 64) - 1) for w in range(words)] for m in bits]
    return [[w - (1 << 64) if w >> 63 else w for w in row] for row in rows]


def cache_layout(fail, ckv_cache: torch.Tensor, kpe_cache: torch.Tensor) -> tuple:
    """(ckv pointer, page and row stride in bytes, the same of kpe, pages) of the two caches."""
    shape = ckv_cache.shape
    pages = shape[0] if shape else 0
    if pages < 1 or shape != (pages, PAGE_SIZE, DIM_CKV) or kpe_cache.shape != (pages, PAGE_SIZE, DIM_KPE):
        fail(f"ckv_cache must be [pages, {PAGE_SIZE}, {DIM_CKV}] and kpe_cache [pages, {PAGE_SIZE}, {DIM_KPE}] with at "
             f"least one page, got {tuple(shape)} and {tuple(kpe_cache.shape)}")
    if ckv_cache.dtype is not torch.bfloat16 or kpe_cache.dtype is not torch.bfloat16:
        fail(f"ckv_cache and kpe_cache must be bfloat16, got {ckv_cache.dtype} and {kpe_cache.dtype}")
    cp, cr, cc = ckv_cache.stride()
    kp, kr, kc = kpe_cache.stride()
    if pages == 1:  # strides that are never taken
        cp, kp = PAGE_SIZE * cr, PAGE_SIZE * kr
    ckv, kpe = ckv_cache.data_ptr(), kpe_cache.data_ptr()
    if cc != 1 or kc != 1 or cr < DIM_CKV or kr < DIM_KPE or cp < cr or kp < kr or (cp | cr | kp | kr) & 7 or \
            (ckv | kpe) & 15:
        fail(f"ckv_cache and kpe_cache must have contiguous rows, 16-byte aligned (strides {ckv_cache.stride()} and "
             f"{kpe_cache.stride()})")
    return ckv, 2 * cp, 2 * cr, kpe, 2 * kp, 2 * kr, pages


def check_device(fail, **tensors) -> None:
    """Names the tensor that is not where the first one is (called once that is known)."""
    first = next(iter(tensors.values()))
    if not first.is_cuda:
        fail("tensors must be on a CUDA device")
    for name, t in tensors.items():
        if t is not None and t.device != first.device:
            fail(f"{name} is on {t.device}, expected {first.device}")


def check_rows(fail, q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table, cu_drafts, tree_mask) -> tuple:
    """The checks shared with ``dsa_b200.evict.accumulate``; returns the sizes and
    the arguments of the C entry points up to ``mask_words``, and the tensors
    that hold them.  Every message is formatted only on failure: this runs once
    per step and layer, and short contexts wait for the host."""
    at = q_nope.get_device()
    if at < 0 or q_pe.get_device() != at or ckv_cache.get_device() != at or kpe_cache.get_device() != at or \
            prefix_lens.get_device() != at or block_table.get_device() != at or cu_drafts.get_device() != at or \
            tree_mask.get_device() != at:
        check_device(fail, q_nope=q_nope, q_pe=q_pe, ckv_cache=ckv_cache, kpe_cache=kpe_cache, prefix_lens=prefix_lens,
                     block_table=block_table, cu_drafts=cu_drafts, tree_mask=tree_mask)
    shape = q_nope.shape
    if len(shape) != 3 or shape[2] != DIM_CKV or not 1 <= shape[1] <= MAX_HEADS:
        fail(f"q_nope must be [T, heads <= {MAX_HEADS}, {DIM_CKV}], got {tuple(shape)}")
    T, H, _ = shape
    if q_pe.shape != (T, H, DIM_KPE):
        fail(f"q_pe must be [{T}, {H}, {DIM_KPE}]")
    if q_nope.dtype is not torch.bfloat16 or q_pe.dtype is not torch.bfloat16:
        fail(f"q_nope and q_pe must be bfloat16, got {q_nope.dtype} and {q_pe.dtype}")
    caches = cache_layout(fail, ckv_cache, kpe_cache)
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1:
        fail("block_table must be [B, max_pages]")
    B, max_pages = shape
    if prefix_lens.dtype is not torch.int32 or prefix_lens.shape != (B,):
        fail(f"prefix_lens must be int32 [{B}]")
    if cu_drafts.shape != (B + 1,):
        fail(f"cu_drafts must be int32 [{B + 1}] (one more than block_table rows)")
    shape = tree_mask.shape
    if tree_mask.dtype is not torch.int64 or len(shape) != 2 or shape[0] != T or not 1 <= shape[1] <= MAX_MASK_WORDS:
        fail(f"tree_mask must be int64 [{T}, words <= {MAX_MASK_WORDS}]")
    if T * H > 1 << 24 or B > 65536 or (T * H // 64 + B) * (max_pages + 3) > 1 << 30:
        fail(f"{T} drafts of {H} heads over {B} requests of {max_pages} pages are more than one call takes")
    qn = q_nope if q_nope.is_contiguous() else q_nope.contiguous()
    qp = q_pe if q_pe.is_contiguous() else q_pe.contiguous()
    pl = prefix_lens if prefix_lens.is_contiguous() else prefix_lens.contiguous()
    tm = tree_mask if tree_mask.is_contiguous() else tree_mask.contiguous()
    bt, cu = int32_of("block_table", block_table, fail), int32_of("cu_drafts", cu_drafts, fail)
    args = (qn.data_ptr(), qp.data_ptr(), *caches, pl.data_ptr(), bt.data_ptr(), cu.data_ptr(), tm.data_ptr(), B, T, H,
            max_pages, shape[1])
    return at, T, H, B, max_pages, args, (qn, qp, pl, bt, cu, tm)


def int32_of(name: str, t: torch.Tensor, fail) -> torch.Tensor:
    if t.dtype is not torch.int32:
        if t.dtype is not torch.int64:
            fail(f"{name} must be int32 or int64")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _fail(msg: str) -> None:
    raise ValueError(f"dsa_tree.run: {msg}")


def _workspace_bytes(dev: torch.device) -> int:
    n = _ws_bytes.get(dev.index)
    if n is None:
        n = _ws_bytes[dev.index] = _native.call_on(dev, _native.lib().dsa_tree_attention_workspace_bytes)
    return n


def run(q_nope: torch.Tensor, q_pe: torch.Tensor, ckv_cache: torch.Tensor, kpe_cache: torch.Tensor,
        prefix_lens: torch.Tensor, block_table: torch.Tensor, cu_drafts: torch.Tensor, tree_mask: torch.Tensor,
        sm_scale, output: torch.Tensor, lse: torch.Tensor) -> None:
    at, T, H, B, _, args, hold = check_rows(_fail, q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table,
                                            cu_drafts, tree_mask)
    if output.get_device() != at or lse.get_device() != at:
        check_device(_fail, q_nope=q_nope, output=output, lse=lse)
    if output.dtype is not torch.bfloat16 or output.shape != (T, H, DIM_CKV) or not output.is_contiguous():
        _fail(f"output must be contiguous bfloat16 [{T}, {H}, {DIM_CKV}]")
    if lse.dtype is not torch.float32 or lse.shape != (T, H) or not lse.is_contiguous():
        _fail(f"lse must be contiguous float32 [{T}, {H}]")
    sm_scale = float(sm_scale)
    if T == 0 or B == 0:
        return
    dev = q_nope.device
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "tree", _workspace_bytes(dev), cur)
    st = _native.call_on(dev, _native.lib().dsa_tree_attention_run, *args, sm_scale, output.data_ptr(), lse.data_ptr(),
                         ws.data_ptr(), ws.numel(), cur)
    if st:
        if st == _native.DSA_ERR_OVERLAP:
            _fail("output and lse must share memory neither with each other nor with the inputs (output may be q_nope itself)")
        _native.check(st, "dsa_tree_attention_run")
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        raise_on_device_status(dev)


def device_status(device: torch.device, clear: bool = True) -> int:
    """OR of the sticky device status bits of every tree attention workspace on
    `device` (synchronises)."""
    return read_status(device, "tree", clear)


def read_status(device: torch.device, name: str, clear: bool) -> int:
    bits = 0
    stream = ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)
    for ws in workspace.buffers_of(device, name):
        out = ctypes.c_uint32(0)
        with torch.cuda.device(device):
            st = _native.lib().dsa_read_device_status(ctypes.c_void_p(ws.data_ptr()), ctypes.byref(out),
                                                      int(clear), stream)
        _native.check(st, "dsa_read_device_status")
        bits |= int(out.value)
    return bits


def raise_on_device_status(device: torch.device) -> None:
    bits = device_status(device, clear=True)
    if bits:
        raise _native.DsaError(f"dsa_tree: {_native.describe_device_status(bits)} (status bits {bits:#x})")
