"""The paged latent cache in 8 bits (destination-passing style): written with
the latent's norm and the position part's rotation in one pass, read back as
bf16 rows, and attended to.

    write(kv, slot_mapping, latent_cache, norm_weight=None, eps=1e-6,
          positions=None, cos_sin=None, interleaved=False) -> None
    read(latent_cache, block_table, starts, cu_rows, ckv, kpe) -> None
    attend(q_nope, q_pe, latent_cache, seq_lens, block_table, cu_rows, sm_scale,
           output, lse) -> None
    attend_sparse(q_nope, q_pe, latent_cache, sparse_indices, sm_scale, output,
                  lse) -> None

``latent_cache`` takes the place of the bf16 ``ckv`` / ``kpe`` caches that
``dsa_b200.attention`` and ``dsa_b200.tree`` read, at 644 bytes a token for 1152:
pages of 41216 bytes (``PAGE_BYTES``; a contiguous 1-byte tensor of any shape)
hold 64 x 512 float8_e4m3fn codes, 64 x 64 bf16 of the position part and 64
float32 scales, one for each token, whose latent is code * scale.  Slots and
block tables are those of the other caches.

``write`` takes rows ``[N, 576]`` as a projection gives them (rows may be
strided): the first 512 values c become
    codes e4m3(448 t / max|t|) of t = c * norm_weight, and the scale
    max|t| / 448 / sqrt(mean(c^2) + eps),
the last 64 are rotated by their position's 32 angles (``cos_sin``: [positions,
64] float32, cosines then sines; pairs (i, i + 32), or (2 i, 2 i + 1) with
``interleaved``) and rounded to bf16.  Without ``norm_weight`` the latent is
stored as given, without ``cos_sin`` the position part.  Negative slots are
padding and skipped; a slot beyond the cache or a position beyond the table
sets a status bit, and the token is not written.  A slot given twice in a call
holds either of its tokens, or parts of both.  A latent with an infinity or NaN,
or whose scale would be above float32's largest number, is stored as NaN
throughout; one whose scale would be below 2^-126 as zeros (both with scale 1).

``read`` makes row ``cu_rows[r] + i`` of ``ckv`` [T, 512] and ``kpe`` [T, 64]
(bf16, rows may be strided, such as the two parts of one [T, 576] buffer) the
token at position ``starts[r] + i`` of request r.  Rows outside of
``[cu_rows[0], cu_rows[-1])`` are left as they are; a row whose position or page
does not exist is zeros and sets a status bit.

``attend`` reads everything a request has cached, as ``dsa_b200.tree.run`` does
of the bf16 caches: with ``cu_rows`` None one row per request (plain decoding);
else request r has the rows ``cu_rows[r] .. cu_rows[r+1]-1`` of ``q_nope`` / ``q_pe``,
its last tokens (a chain of drafts, written to the cache before), and row j of n
sees the first ``seq_lens[r] - n + 1 + j`` tokens.  ``attend_sparse`` reads the slots
of ``sparse_indices`` [T, K] (-1: none; a slot given twice counts twice), as
``dsa_b200.attention.run`` does.  Both take 1 to 128 heads; ``lse`` is the base-2 log-sum-exp of the scaled logits; a row that
sees nothing yields output 0 and lse -inf.  Tokens that no row sees may hold
anything; a visible one with NaN makes the output NaN.  ``output`` may be ``q_nope``
itself; other outputs over an input are refused.  Values of a query are exact from
2^-13 of its row's largest up, smaller ones to 2^-21 of that; softmax weights times
scales to 2^-14 of each and 2^-28 of the row's largest.  Where scales of one request
differ by 2^60 and more, tokens of the small ones may count as zeros.

Calls that overlap need different streams; threads may call on one stream.  A
captured graph uses the workspace of the stream that it was captured on: it must
not run beside another one captured there, nor beside calls on that stream.
Launches go to the current stream and can be captured into a CUDA graph (make
one call on the capturing stream first).  ``device_status`` reads the sticky
status bits; with ``DSA_B200_CHECK=1`` each call synchronises and raises.
"""

from __future__ import annotations

import os

import torch

from . import _native, workspace
from .tree import check_device, int32_of, read_status

PAGE_SIZE = 64
DIM_CKV = 512
DIM_KPE = 64
MAX_HEADS = 128
PAGE_BYTES = PAGE_SIZE * (DIM_CKV + 2 * DIM_KPE + 4)

_CHECK = os.environ.get("DSA_B200_CHECK", "0") not in ("", "0")
_ws_bytes: dict = {}  # device index -> dsa_latent_attention_workspace_bytes


def _fail_write(msg: str) -> None:
    raise ValueError(f"dsa_quant.write: {msg}")


def _fail_read(msg: str) -> None:
    raise ValueError(f"dsa_quant.read: {msg}")


def _fail_attend(msg: str) -> None:
    raise ValueError(f"dsa_quant.attend: {msg}")


def _fail_sparse(msg: str) -> None:
    raise ValueError(f"dsa_quant.attend_sparse: {msg}")


def _pages(fail, latent_cache: torch.Tensor) -> int:
    nbytes = latent_cache.numel()
    if latent_cache.element_size() != 1 or not latent_cache.is_contiguous() or nbytes % PAGE_BYTES or nbytes == 0:
        fail(f"latent_cache must be a contiguous 1-byte tensor of pages of {PAGE_BYTES} bytes, at least one")
    if latent_cache.data_ptr() & 15:
        fail("latent_cache must be 16-byte aligned")
    return nbytes // PAGE_BYTES


def _rows(fail, name: str, t: torch.Tensor, rows, width: int) -> int:
    """Bytes from row to row of a bf16 [rows, width] tensor."""
    shape = t.shape
    if t.dtype is not torch.bfloat16 or len(shape) != 2 or shape[1] != width or (rows is not None and shape[0] != rows):
        fail(f"{name} must be bfloat16 [{'N' if rows is None else rows}, {width}], got {t.dtype} {tuple(shape)}")
    pitch, step = t.stride()
    if shape[0] <= 1:
        pitch = width
    if (step != 1 and width > 1) or pitch < width or pitch & 7 or t.data_ptr() & 15:
        fail(f"{name} must have contiguous rows, 16-byte aligned (strides {t.stride()})")
    return 2 * pitch


def _int64_of(fail, name: str, t: torch.Tensor, n: int) -> torch.Tensor:
    if t.shape != (n,) or t.dtype not in (torch.int64, torch.int32):
        fail(f"{name} must be int64 or int32 [{n}]")
    if t.dtype is not torch.int64:
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def _finish(status: int, entry: str, fail, dev: torch.device) -> None:
    if status:
        if status == _native.DSA_ERR_OVERLAP:
            fail("what is written must share memory neither with an input nor with another output")
        _native.check(status, entry)
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        raise_on_device_status(dev)


def write(kv: torch.Tensor, slot_mapping: torch.Tensor, latent_cache: torch.Tensor, norm_weight: torch.Tensor = None,
          eps: float = 1e-6, positions: torch.Tensor = None, cos_sin: torch.Tensor = None,
          interleaved: bool = False) -> None:
    at = kv.get_device()
    if at < 0 or slot_mapping.get_device() != at or latent_cache.get_device() != at or \
            any(t is not None and t.get_device() != at for t in (norm_weight, positions, cos_sin)):
        check_device(_fail_write, kv=kv, slot_mapping=slot_mapping, latent_cache=latent_cache, norm_weight=norm_weight,
                     positions=positions, cos_sin=cos_sin)
    pitch = _rows(_fail_write, "kv", kv, None, DIM_CKV + DIM_KPE)
    n = kv.shape[0]
    slots = _int64_of(_fail_write, "slot_mapping", slot_mapping, n)
    pages = _pages(_fail_write, latent_cache)
    norm = 0
    if norm_weight is not None:
        if norm_weight.dtype is not torch.bfloat16 or norm_weight.shape != (DIM_CKV,) or not norm_weight.is_contiguous() or \
                norm_weight.data_ptr() & 15:
            _fail_write(f"norm_weight must be contiguous bfloat16 [{DIM_CKV}], 16-byte aligned")
        norm = norm_weight.data_ptr()
    if (positions is None) != (cos_sin is None):
        _fail_write("positions and cos_sin come together")
    pos, angles, most = None, 0, 0
    if positions is not None:
        pos = _int64_of(_fail_write, "positions", positions, n)
        if cos_sin.dtype is not torch.float32 or cos_sin.dim() != 2 or cos_sin.shape[1] != DIM_KPE or cos_sin.shape[0] < 1 or \
                not cos_sin.is_contiguous() or cos_sin.data_ptr() & 7:
            _fail_write(f"cos_sin must be contiguous float32 [positions, {DIM_KPE}]")
        angles, most = cos_sin.data_ptr(), cos_sin.shape[0]
    if n >= 1 << 31:
        _fail_write(f"{n} tokens are more than one call takes")
    if n == 0:
        return
    dev = kv.device
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "quant_rows", _native.WORKSPACE_HEADER, cur)
    st = _native.call_on(dev, _native.lib().dsa_latent_cache_write, kv.data_ptr(), pitch, slots.data_ptr(), n, norm,
                         float(eps), pos.data_ptr() if pos is not None else 0, angles, most, int(bool(interleaved)),
                         latent_cache.data_ptr(), pages, ws.data_ptr(), cur)
    _finish(st, "dsa_latent_cache_write", _fail_write, dev)


def read(latent_cache: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, cu_rows: torch.Tensor,
         ckv: torch.Tensor, kpe: torch.Tensor) -> None:
    at = latent_cache.get_device()
    if at < 0 or block_table.get_device() != at or starts.get_device() != at or cu_rows.get_device() != at or \
            ckv.get_device() != at or kpe.get_device() != at:
        check_device(_fail_read, latent_cache=latent_cache, block_table=block_table, starts=starts, cu_rows=cu_rows,
                     ckv=ckv, kpe=kpe)
    pages = _pages(_fail_read, latent_cache)
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1:
        _fail_read("block_table must be [B, max_pages]")
    B, max_pages = shape
    if starts.shape != (B,) or cu_rows.shape != (B + 1,):
        _fail_read(f"starts must be [{B}] and cu_rows [{B + 1}]")
    ckv_pitch = _rows(_fail_read, "ckv", ckv, None, DIM_CKV)
    T = ckv.shape[0]
    kpe_pitch = _rows(_fail_read, "kpe", kpe, T, DIM_KPE)
    bt, st, cu = (int32_of(name, t, _fail_read) for name, t in
                  (("block_table", block_table), ("starts", starts), ("cu_rows", cu_rows)))
    if T >= 1 << 31:
        _fail_read(f"{T} rows are more than one call takes")
    if T == 0 or B == 0:
        return
    dev = latent_cache.device
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "quant_rows", _native.WORKSPACE_HEADER, cur)
    status = _native.call_on(dev, _native.lib().dsa_latent_cache_read, latent_cache.data_ptr(), pages, bt.data_ptr(),
                             st.data_ptr(), cu.data_ptr(), B, max_pages, T, ckv.data_ptr(), ckv_pitch, kpe.data_ptr(),
                             kpe_pitch, ws.data_ptr(), cur)
    _finish(status, "dsa_latent_cache_read", _fail_read, dev)


def _queries(fail, q_nope, q_pe, output, lse) -> tuple:
    shape = q_nope.shape
    if len(shape) != 3 or shape[2] != DIM_CKV or not 1 <= shape[1] <= MAX_HEADS:
        fail(f"q_nope must be [T, heads <= {MAX_HEADS}, {DIM_CKV}], got {tuple(shape)}")
    T, H, _ = shape
    if q_pe.shape != (T, H, DIM_KPE):
        fail(f"q_pe must be [{T}, {H}, {DIM_KPE}]")
    if q_nope.dtype is not torch.bfloat16 or q_pe.dtype is not torch.bfloat16:
        fail(f"q_nope and q_pe must be bfloat16, got {q_nope.dtype} and {q_pe.dtype}")
    if output.dtype is not torch.bfloat16 or output.shape != shape or not output.is_contiguous():
        fail(f"output must be contiguous bfloat16 [{T}, {H}, {DIM_CKV}]")
    if lse.dtype is not torch.float32 or lse.shape != (T, H) or not lse.is_contiguous():
        fail(f"lse must be contiguous float32 [{T}, {H}]")
    if T * H > 1 << 24:
        fail(f"{T} rows of {H} heads are more than one call takes")
    return T, H, q_nope if q_nope.is_contiguous() else q_nope.contiguous(), q_pe if q_pe.is_contiguous() else q_pe.contiguous()


def _workspace(dev: torch.device, cur: int) -> torch.Tensor:
    n = _ws_bytes.get(dev.index)
    if n is None:
        n = _ws_bytes[dev.index] = _native.call_on(dev, _native.lib().dsa_latent_attention_workspace_bytes)
    return workspace.get(dev, "quant", n, cur)


def attend(q_nope: torch.Tensor, q_pe: torch.Tensor, latent_cache: torch.Tensor, seq_lens: torch.Tensor,
           block_table: torch.Tensor, cu_rows, sm_scale, output: torch.Tensor, lse: torch.Tensor) -> None:
    at = q_nope.get_device()
    if at < 0 or q_pe.get_device() != at or latent_cache.get_device() != at or seq_lens.get_device() != at or \
            block_table.get_device() != at or (cu_rows is not None and cu_rows.get_device() != at) or \
            output.get_device() != at or lse.get_device() != at:
        check_device(_fail_attend, q_nope=q_nope, q_pe=q_pe, latent_cache=latent_cache, seq_lens=seq_lens,
                     block_table=block_table, cu_rows=cu_rows, output=output, lse=lse)
    T, H, qn, qp = _queries(_fail_attend, q_nope, q_pe, output, lse)
    pages = _pages(_fail_attend, latent_cache)
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1:
        _fail_attend("block_table must be [B, max_pages]")
    B, max_pages = shape
    if seq_lens.shape != (B,):
        _fail_attend(f"seq_lens must be int32 [{B}]")
    if cu_rows is None:
        if T != B:
            _fail_attend(f"without cu_rows there is one row for each of the {B} requests, not {T}")
    elif cu_rows.shape != (B + 1,):
        _fail_attend(f"cu_rows must be int32 [{B + 1}] (one more than block_table rows)")
    if B > 65536 or (T * H // 16 + B) * (max_pages // 2 + 4) > 1 << 30:
        _fail_attend(f"{T} rows of {H} heads over {B} requests of {max_pages} pages are more than one call takes")
    bt, sl = int32_of("block_table", block_table, _fail_attend), int32_of("seq_lens", seq_lens, _fail_attend)
    cu = int32_of("cu_rows", cu_rows, _fail_attend) if cu_rows is not None else None
    sm_scale = float(sm_scale)
    if T == 0 or B == 0:
        return
    dev = q_nope.device
    cur = _native.current_stream(dev)
    ws = _workspace(dev, cur)
    st = _native.call_on(dev, _native.lib().dsa_latent_attention_run, qn.data_ptr(), qp.data_ptr(), latent_cache.data_ptr(),
                         pages, sl.data_ptr(), bt.data_ptr(), cu.data_ptr() if cu is not None else 0, B, T, H, max_pages,
                         sm_scale, output.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(), cur)
    _finish(st, "dsa_latent_attention_run", _fail_attend, dev)


def attend_sparse(q_nope: torch.Tensor, q_pe: torch.Tensor, latent_cache: torch.Tensor, sparse_indices: torch.Tensor,
                  sm_scale, output: torch.Tensor, lse: torch.Tensor) -> None:
    at = q_nope.get_device()
    if at < 0 or q_pe.get_device() != at or latent_cache.get_device() != at or sparse_indices.get_device() != at or \
            output.get_device() != at or lse.get_device() != at:
        check_device(_fail_sparse, q_nope=q_nope, q_pe=q_pe, latent_cache=latent_cache, sparse_indices=sparse_indices,
                     output=output, lse=lse)
    T, H, qn, qp = _queries(_fail_sparse, q_nope, q_pe, output, lse)
    pages = _pages(_fail_sparse, latent_cache)
    shape = sparse_indices.shape
    if len(shape) != 2 or shape[0] != T or not 1 <= shape[1] <= 65536:
        _fail_sparse(f"sparse_indices must be [{T}, 1 to 65536]")
    if T * ((H + 15) // 16) > 1 << 20:
        _fail_sparse(f"{T} rows of {H} heads over {shape[1]} slots are more than one call takes")
    if pages > 0x7FFFFFFF // PAGE_SIZE:
        _fail_sparse("latent_cache has more slots than an index can name")
    idx = int32_of("sparse_indices", sparse_indices, _fail_sparse)
    sm_scale = float(sm_scale)
    if T == 0:
        return
    dev = q_nope.device
    cur = _native.current_stream(dev)
    ws = _workspace(dev, cur)
    st = _native.call_on(dev, _native.lib().dsa_latent_sparse_attention_run, qn.data_ptr(), qp.data_ptr(),
                         latent_cache.data_ptr(), pages, idx.data_ptr(), T, H, shape[1], sm_scale, output.data_ptr(),
                         lse.data_ptr(), ws.data_ptr(), ws.numel(), cur)
    _finish(st, "dsa_latent_sparse_attention_run", _fail_sparse, dev)


def device_status(device: torch.device, clear: bool = True) -> int:
    """OR of the sticky status bits of every workspace of these operators on
    `device` (synchronises)."""
    return read_status(device, "quant_rows", clear) | read_status(device, "quant", clear)


def raise_on_device_status(device: torch.device) -> None:
    bits = device_status(device, clear=True)
    if bits:
        raise _native.DsaError(f"dsa_quant: {_native.describe_device_status(bits)} (status bits {bits:#x})")
