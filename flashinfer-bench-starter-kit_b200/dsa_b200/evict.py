"""Eviction from the paged caches by accumulated attention weight
(destination-passing style).

    accumulate(q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table,
               cu_drafts, tree_mask, sm_scale, lse, acc, out) -> None

The attention weight that every cached token got from the rows of a
``dsa_b200.tree.run`` with the same arguments (``lse`` is what that call gave),
summed over its rows and heads and added to the token's accumulator:

    out[r, k] = acc[r, k] + sum over drafts i of request r and heads h that see
                position k of 2^(scaled logit - lse[i, h])

``acc`` and ``out`` are float32 ``[B, max_pages * 64]`` by position in the
request (not by cache slot, so requests that share pages keep sums of their
own); ``out`` may be ``acc``.  Every element of ``out`` is written.  To count
accepted drafts only, pass their rows alone, with a ``cu_drafts`` and masks to
match.  The sums run in a fixed order, so that results repeat.
"""

from __future__ import annotations

import torch

from . import _native, tree, workspace

PAGE_SIZE = 64


def _fail_acc(msg: str) -> None:
    raise ValueError(f"dsa_evict.accumulate: {msg}")


def _rows_of(name: str, t: torch.Tensor, shape: tuple, fail) -> None:
    if t.dtype != torch.float32 or tuple(t.shape) != shape:
        fail(f"{name} must be float32 {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.stride(1) != 1 or (shape[0] > 1 and t.stride(0) < shape[1]):
        fail(f"{name} must have contiguous rows that do not overlap (strides {t.stride()})")


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def accumulate(q_nope: torch.Tensor, q_pe: torch.Tensor, ckv_cache: torch.Tensor, kpe_cache: torch.Tensor,
               prefix_lens: torch.Tensor, block_table: torch.Tensor, cu_drafts: torch.Tensor,
               tree_mask: torch.Tensor, sm_scale, lse: torch.Tensor, acc: torch.Tensor, out: torch.Tensor) -> None:
    dev, T, H, B, max_pages, args, hold = tree.check_rows(
        _fail_acc, q_nope, q_pe, ckv_cache, kpe_cache, prefix_lens, block_table, cu_drafts, tree_mask,
        (("lse", lse), ("acc", acc), ("out", out)))
    if lse.dtype != torch.float32 or lse.shape != (T, H):
        _fail_acc(f"lse must be float32 [{T}, {H}]")
    _rows_of("acc", acc, (B, max_pages * PAGE_SIZE), _fail_acc)
    _rows_of("out", out, (B, max_pages * PAGE_SIZE), _fail_acc)
    same = acc.data_ptr() == out.data_ptr()
    if same and _pitch(acc) != _pitch(out):
        _fail_acc("acc and out overlap")
    if isinstance(sm_scale, torch.Tensor):
        sm_scale = float(sm_scale.item())
    if B == 0:
        return
    if T == 0:
        if not same:
            out.copy_(acc)
        return
    lse = lse.contiguous()
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "evict", _native.WORKSPACE_HEADER, cur)
    st = _native.call_on(dev, _native.lib().dsa_tree_weights_run, *args, float(sm_scale), lse.data_ptr(),
                         acc.data_ptr(), _pitch(acc), out.data_ptr(), _pitch(out), ws.data_ptr(), ws.numel(), cur)
    _native.check(st, "dsa_tree_weights_run")
    if tree._CHECK and not torch.cuda.is_current_stream_capturing():
        raise_on_device_status(dev)


def device_status(device: torch.device, clear: bool = True) -> int:
    """OR of the sticky device status bits of every eviction workspace on
    `device` (synchronises)."""
    return tree.read_status(device, "evict", clear)


def raise_on_device_status(device: torch.device) -> None:
    bits = device_status(device, clear=True)
    if bits:
        raise _native.DsaError(f"dsa_evict: {_native.describe_device_status(bits)} (status bits {bits:#x})")
