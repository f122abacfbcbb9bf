"""Eviction from the paged caches by accumulated attention weight
(destination-passing style).

    accumulate(q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table,
               cu_drafts, tree_mask, sm_scale, lse, acc, out) -> None
    run(acc, seq_lens, block_table, new_block_table, ckv_cache, kpe_cache,
        k_index_cache_fp8, num_sink, num_recent, keep, new_seq_lens, new_acc) -> None

``accumulate``: the attention weight that every cached token got from the rows of a
``dsa_b200.tree.run`` with the same arguments (``lse`` is what that call gave),
summed over its rows and heads and added to the token's accumulator:

    out[r, k] = acc[r, k] + sum over drafts i of request r and heads h that see
                position k of 2^(scaled logit - lse[i, h])

``acc`` and ``out`` are float32 ``[B, max_pages * 64]`` by position in the
request (not by cache slot, so requests that share pages keep sums of their
own); ``out`` may be ``acc``.  Every element of ``out`` is written.  The sums run
in a fixed order, so that results repeat.

To count accepted drafts only, give the others' rows an ``lse`` of -inf, for
example ``lse.masked_fill(~accepted[:, None], -math.inf)``: such a row adds
nothing.  (Leaving the rows out is another call: a draft's position is its
place among its request's rows, so that accepted drafts 0 and 3 passed alone
would be taken for the drafts at positions prefix and prefix + 1.)

``run``: a request with more than ``budget = keep.shape[1]`` tokens keeps its
first ``num_sink``, its last ``num_recent`` and, of the tokens between them, those
of largest ``acc`` (equal: the earlier; NaN is largest), ``budget`` in all; the
others keep everything.  What is kept stays in order: position ``keep[r, i]``
(ascending, then -1) becomes position i of ``new_block_table``'s row, in the ckv
and kpe caches and, unless it is None, in the indexer's FP8 key cache.
``new_seq_lens`` (which may be ``seq_lens`` itself) and ``new_acc`` (float32
``[B, new_max_pages * 64]``, 0 behind the kept tokens) go with the new table.

The new pages are pages of the same pool that no row of ``block_table`` uses; the
old ones are not changed, so requests may share them, and the caller frees
them.  With ``DSA_B200_CHECK=1`` a call whose new pages are also old ones, or
given twice, raises.  Streams, graphs and device status bits are as for
``dsa_b200.tree``.
"""

from __future__ import annotations

import operator

import torch

from . import _native, tree, workspace

PAGE_SIZE = 64
INDEX_PAGE_BYTES = PAGE_SIZE * 128 + PAGE_SIZE * 4


def _fail_acc(msg: str) -> None:
    raise ValueError(f"dsa_evict.accumulate: {msg}")


def _rows_of(name: str, t: torch.Tensor, rows: int, width: int, fail) -> int:
    """The pitch of a float32 [rows, width] tensor, in elements."""
    if t.dtype is not torch.float32 or t.shape != (rows, width):
        fail(f"{name} must be float32 [{rows}, {width}], got {t.dtype} {tuple(t.shape)}")
    pitch, col = t.stride()
    if col != 1 or (rows > 1 and pitch < width):
        fail(f"{name} must have contiguous rows that do not overlap (strides {t.stride()})")
    return pitch if rows > 1 else width


def _overlap(rows: int, a: int, a_pitch: int, a_width: int, b: int, b_pitch: int, b_width: int) -> bool:
    """Whether two float32 tensors of `rows` contiguous rows at the addresses a
    and b (pitches and widths in elements) share memory."""
    if a > b:
        a, a_pitch, a_width, b, b_pitch, b_width = b, b_pitch, b_width, a, a_pitch, a_width
    apart = (b - a) // 4
    if apart >= (rows - 1) * a_pitch + a_width:
        return False
    # Interleaved rows of one buffer, such as its left and right columns.
    at = apart % a_pitch
    return a_pitch != b_pitch or at < a_width or at + b_width > a_pitch


def accumulate(q_nope: torch.Tensor, q_pe: torch.Tensor, ckv_cache: torch.Tensor, kpe_cache: torch.Tensor,
               prefix_lens: torch.Tensor, block_table: torch.Tensor, cu_drafts: torch.Tensor,
               tree_mask: torch.Tensor, sm_scale, lse: torch.Tensor, acc: torch.Tensor, out: torch.Tensor) -> None:
    at, T, H, B, max_pages, args, hold = tree.check_rows(
        _fail_acc, q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table, cu_drafts, tree_mask)
    if lse.get_device() != at or acc.get_device() != at or out.get_device() != at:
        tree.check_device(_fail_acc, q_nope=q_nope, lse=lse, acc=acc, out=out)
    if lse.dtype is not torch.float32 or lse.shape != (T, H):
        _fail_acc(f"lse must be float32 [{T}, {H}]")
    width = max_pages * PAGE_SIZE
    acc_pitch, out_pitch = _rows_of("acc", acc, B, width, _fail_acc), _rows_of("out", out, B, width, _fail_acc)
    acc_ptr, out_ptr = acc.data_ptr(), out.data_ptr()
    same = acc_ptr == out_ptr and acc_pitch == out_pitch
    if not same and B > 0 and _overlap(B, acc_ptr, acc_pitch, width, out_ptr, out_pitch, width):
        _fail_acc("out must be acc itself or not overlap it")
    sm_scale = float(sm_scale)
    if B == 0:
        return
    if T == 0:
        if not same:
            out.copy_(acc)
        return
    if not lse.is_contiguous():
        lse = lse.contiguous()
    dev = q_nope.device
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "evict", _native.WORKSPACE_HEADER, cur)
    st = _native.call_on(dev, _native.lib().dsa_tree_weights_run, *args, sm_scale, lse.data_ptr(), acc_ptr, acc_pitch,
                         out_ptr, out_pitch, ws.data_ptr(), ws.numel(), cur)
    if st:
        if st == _native.DSA_ERR_OVERLAP:
            _fail_acc("out must share memory with no input but acc, which it may be")
        _native.check(st, "dsa_tree_weights_run")
    if tree._CHECK and not torch.cuda.is_current_stream_capturing():
        raise_on_device_status(dev)


def _fail_run(msg: str) -> None:
    raise ValueError(f"dsa_evict.run: {msg}")


def run(acc: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, new_block_table: torch.Tensor,
        ckv_cache: torch.Tensor, kpe_cache: torch.Tensor, k_index_cache_fp8, num_sink: int, num_recent: int,
        keep: torch.Tensor, new_seq_lens: torch.Tensor, new_acc: torch.Tensor) -> None:
    # Every message is formatted only on failure: small batches wait for the host.
    at = acc.get_device()
    if at < 0 or seq_lens.get_device() != at or block_table.get_device() != at or new_block_table.get_device() != at or \
            ckv_cache.get_device() != at or kpe_cache.get_device() != at or keep.get_device() != at or \
            new_seq_lens.get_device() != at or new_acc.get_device() != at or \
            (k_index_cache_fp8 is not None and k_index_cache_fp8.get_device() != at):
        tree.check_device(_fail_run, acc=acc, seq_lens=seq_lens, block_table=block_table, new_block_table=new_block_table,
                          ckv_cache=ckv_cache, kpe_cache=kpe_cache, k_index_cache_fp8=k_index_cache_fp8, keep=keep,
                          new_seq_lens=new_seq_lens, new_acc=new_acc)
    if len(block_table.shape) != 2 or block_table.shape[1] < 1:
        _fail_run("block_table must be [B, max_pages]")
    B, max_pages = block_table.shape
    if len(new_block_table.shape) != 2 or new_block_table.shape[0] != B or new_block_table.shape[1] < 1:
        _fail_run(f"new_block_table must be [{B}, new_max_pages]")
    new_pages = new_block_table.shape[1]
    caches = tree.cache_layout(_fail_run, ckv_cache, kpe_cache)
    pages = caches[-1]
    if k_index_cache_fp8 is not None:
        if k_index_cache_fp8.element_size() != 1 or not k_index_cache_fp8.is_contiguous():
            _fail_run("k_index_cache_fp8 must be a contiguous 1-byte tensor (written in place)")
        if k_index_cache_fp8.numel() != pages * INDEX_PAGE_BYTES:
            _fail_run(f"k_index_cache_fp8 holds {k_index_cache_fp8.numel()} bytes, not {pages} pages of {INDEX_PAGE_BYTES}")
        if k_index_cache_fp8.data_ptr() % 16:
            _fail_run("k_index_cache_fp8 must be 16-byte aligned")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,):
        _fail_run(f"seq_lens must be int32 [{B}]")
    if new_seq_lens.dtype != torch.int32 or new_seq_lens.shape != (B,) or not new_seq_lens.is_contiguous():
        _fail_run(f"new_seq_lens must be contiguous int32 [{B}]")
    if keep.dtype != torch.int32 or keep.dim() != 2 or keep.shape[0] != B or not keep.is_contiguous():
        _fail_run(f"keep must be contiguous int32 [{B}, budget]")
    budget = keep.shape[1]
    if not 1 <= budget <= new_pages * PAGE_SIZE:
        _fail_run(f"a budget of {budget} tokens (keep.shape[1]) does not fit new_block_table's {new_pages} pages")
    num_sink, num_recent = operator.index(num_sink), operator.index(num_recent)
    if num_sink < 0 or num_recent < 0 or num_sink + num_recent > budget:
        _fail_run(f"num_sink {num_sink} and num_recent {num_recent} must fit the budget of {budget}")
    width, new_width = max_pages * PAGE_SIZE, new_pages * PAGE_SIZE
    acc_pitch = _rows_of("acc", acc, B, width, _fail_run)
    new_pitch = _rows_of("new_acc", new_acc, B, new_width, _fail_run)
    acc_ptr, new_ptr = acc.data_ptr(), new_acc.data_ptr()
    if B > 0 and _overlap(B, acc_ptr, acc_pitch, width, new_ptr, new_pitch, new_width):
        _fail_run("new_acc must not overlap acc")
    if B == 0:
        return
    if B > 65536 or max_pages > 1 << 24 or new_pages > 1 << 24:
        _fail_run(f"{B} requests of {max_pages} pages are more than one call takes")
    sl = seq_lens if seq_lens.is_contiguous() else seq_lens.contiguous()
    bt = tree.int32_of("block_table", block_table, _fail_run)
    nbt = tree.int32_of("new_block_table", new_block_table, _fail_run)
    dev = acc.device
    check = tree._CHECK and not torch.cuda.is_current_stream_capturing()
    if check:
        _check_new_pages(sl, bt, nbt, budget, pages)
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "evict", _native.WORKSPACE_HEADER, cur)
    st = _native.call_on(dev, _native.lib().dsa_cache_evict_run, acc_ptr, acc_pitch, sl.data_ptr(), bt.data_ptr(),
                         nbt.data_ptr(), B, max_pages, new_pages, *caches[:6],
                         None if k_index_cache_fp8 is None else k_index_cache_fp8.data_ptr(), pages, budget, num_sink,
                         num_recent, keep.data_ptr(), new_seq_lens.data_ptr(), new_ptr, new_pitch, ws.data_ptr(),
                         ws.numel(), cur)
    if st:
        if st == _native.DSA_ERR_OVERLAP:
            _fail_run("keep, new_seq_lens and new_acc must share memory neither with one another nor with the inputs "
                      "(new_seq_lens may be seq_lens itself)")
        _native.check(st, "dsa_cache_evict_run")
    if check:
        raise_on_device_status(dev)


def _check_new_pages(seq_lens, block_table, new_block_table, budget: int, pages: int) -> None:
    """Raises if a page to be written is one that is read, or is given twice (synchronises)."""
    def used(lens, table):
        need = (lens.long().clamp(0, table.shape[1] * PAGE_SIZE) + PAGE_SIZE - 1) // PAGE_SIZE
        ids = table[torch.arange(table.shape[1], device=table.device) < need[:, None]].long()
        return torch.bincount(ids[(ids >= 0) & (ids < pages)], minlength=pages)

    old, new = used(seq_lens, block_table), used(seq_lens.clamp(max=budget), new_block_table)
    if bool(((new > 1) | ((new > 0) & (old > 0))).any()):
        raise ValueError("dsa_evict.run: a page of new_block_table is given twice or still in use by block_table")


def device_status(device: torch.device, clear: bool = True) -> int:
    """OR of the sticky device status bits of every eviction workspace on
    `device` (synchronises)."""
    return tree.read_status(device, "evict", clear)


def raise_on_device_status(device: torch.device) -> None:
    bits = device_status(device, clear=True)
    if bits:
        raise _native.DsaError(f"dsa_evict: {_native.describe_device_status(bits)} (status bits {bits:#x})")
