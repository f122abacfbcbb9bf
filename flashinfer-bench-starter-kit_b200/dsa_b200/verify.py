"""Verification of drafted tokens against the target's probabilities, from given
random numbers (speculative decoding; destination-passing style).

    run(target_probs, draft_probs, draft_tokens, parents, cu_drafts, accept_u,
        sample_u, path, num_accepted, next_token) -> None

It follows ``dsa_b200.tree.run`` or ``dsa_b200.quant.attend`` on the same rows:
request r has the rows ``cu_drafts[r] .. cu_drafts[r+1]-1``, of which the first is
its last certain token and every other one a draft; ``parents`` (as
``tree.masks_from_parents`` takes them, -1 for row 0) makes them a tree.  Row i
of ``target_probs`` [T, V] is the target's distribution after row i, row i of
``draft_probs`` the one that the children of row i were drawn from, each by itself.

The walk starts at row 0.  At a row it looks at the children in their order: a
child with token x is accepted if ``accept_u`` of it is below p'(x) / q(x), where
p' is the target's distribution, from which every rejection takes q away (and
normalises what is left).  After an accepted draft it goes on there; where none
is, or at a row without children, ``next_token`` is drawn from p': the first token
whose running sum exceeds ``sample_u[r]`` of the whole.  The tokens are then
distributed as the target's own.  ``path`` [B, W] gets the accepted rows, counted
from the request's first one (0), then -1; ``num_accepted`` their number; a path
that is full ends the walk.

* ``draft_probs=None``: drafts without a distribution of their own (a model's
  likeliest tokens, looked-up ones).  x is accepted with probability p'(x), and a
  rejected one is struck out of p'.
* Probabilities are float32, rows may be strided (the parts of one larger
  buffer); random numbers are float32 in [0, 1).  Distributions are taken as
  summing to 1.  Comparisons and sums are made in 64 bits.
* Where nothing is left of p' (draws that had no probability), the next token is
  drawn from the target's distribution; if that has none either, it is -1.  So it
  is for a request without rows, and where what is drawn from holds NaN: in the
  target's row, or after a rejection in the draft's.  Probabilities are 0 (of
  either sign) or more.
* A token outside of the vocabulary is never accepted and sets a status bit
  (``device_status``), as do ``cu_drafts`` that do not fit (the request is then
  taken as empty) and requests of over 4096 rows (the others are left out).
* Nothing synchronises; launches go to the current stream and can be captured
  into a CUDA graph (make one call on the capturing stream first).
"""

from __future__ import annotations

import os

import torch

from . import _native, workspace
from .tree import check_device, int32_of, read_status

_CHECK = os.environ.get("DSA_B200_CHECK", "0") not in ("", "0")


def _fail(msg: str) -> None:
    raise ValueError(f"dsa_verify.run: {msg}")


def _pitch(name: str, t: torch.Tensor, rows: int, vocab: int) -> int:
    """Values from row to row."""
    pitch, step = t.stride()
    if rows <= 1:
        pitch = max(pitch, vocab)
    if (step != 1 and vocab > 1) or pitch < vocab:
        _fail(f"{name} must have contiguous rows (strides {t.stride()})")
    return pitch


def run(target_probs: torch.Tensor, draft_probs, draft_tokens: torch.Tensor, parents: torch.Tensor,
        cu_drafts: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, path: torch.Tensor,
        num_accepted: torch.Tensor, next_token: torch.Tensor) -> None:
    # Every message is formatted only on failure: this runs once per step, and small batches wait for the host.
    at = target_probs.get_device()
    if at < 0 or (draft_probs is not None and draft_probs.get_device() != at) or draft_tokens.get_device() != at or \
            parents.get_device() != at or cu_drafts.get_device() != at or accept_u.get_device() != at or \
            sample_u.get_device() != at or path.get_device() != at or num_accepted.get_device() != at or \
            next_token.get_device() != at:
        check_device(_fail, target_probs=target_probs, draft_probs=draft_probs, draft_tokens=draft_tokens, parents=parents,
                     cu_drafts=cu_drafts, accept_u=accept_u, sample_u=sample_u, path=path, num_accepted=num_accepted,
                     next_token=next_token)
    shape = target_probs.shape
    if target_probs.dtype is not torch.float32 or len(shape) != 2 or shape[1] < 1:
        _fail(f"target_probs must be float32 [T, V], got {target_probs.dtype} {tuple(shape)}")
    T, V = shape
    pitch = _pitch("target_probs", target_probs, T, V)
    draft, draft_pitch = 0, 0
    if draft_probs is not None:
        if draft_probs.dtype is not torch.float32 or draft_probs.shape != shape:
            _fail(f"draft_probs must be float32 [{T}, {V}], got {draft_probs.dtype} {tuple(draft_probs.shape)}")
        draft, draft_pitch = draft_probs.data_ptr(), _pitch("draft_probs", draft_probs, T, V)
    one = (T,)
    if draft_tokens.shape != one or parents.shape != one:
        _fail(f"draft_tokens and parents must be [{T}]")
    if cu_drafts.dim() != 1 or cu_drafts.shape[0] < 1:
        _fail("cu_drafts must be [B + 1]")
    B = cu_drafts.shape[0] - 1
    each = (B,)
    if accept_u.dtype is not torch.float32 or accept_u.shape != one or sample_u.dtype is not torch.float32 or \
            sample_u.shape != each:
        _fail(f"accept_u must be float32 [{T}] and sample_u float32 [{B}]")
    shape = path.shape
    if path.dtype is not torch.int32 or len(shape) != 2 or shape[0] != B or shape[1] < 1 or not path.is_contiguous():
        _fail(f"path must be contiguous int32 [{B}, at least 1]")
    W = shape[1]
    if num_accepted.dtype is not torch.int32 or num_accepted.shape != each or not num_accepted.is_contiguous() or \
            next_token.dtype is not torch.int32 or next_token.shape != each or not next_token.is_contiguous():
        _fail(f"num_accepted and next_token must be contiguous int32 [{B}]")
    if T > 1 << 24 or B > 65536 or V > 1 << 28 or W > 1 << 16:
        _fail(f"{T} rows of {B} requests over {V} tokens, paths of {W}, are more than one call takes")
    tok, par, cu = (int32_of("draft_tokens", draft_tokens, _fail), int32_of("parents", parents, _fail),
                    int32_of("cu_drafts", cu_drafts, _fail))
    au = accept_u if accept_u.is_contiguous() else accept_u.contiguous()
    su = sample_u if sample_u.is_contiguous() else sample_u.contiguous()
    if B == 0:
        return
    if T == 0:
        path.fill_(-1)
        num_accepted.zero_()
        next_token.fill_(-1)
        return
    dev = target_probs.device
    cur = _native.current_stream(dev)
    ws = workspace.get(dev, "verify", _native.WORKSPACE_HEADER, cur)
    st = _native.call_on(dev, _native.lib().dsa_verify_run, target_probs.data_ptr(), pitch, draft, draft_pitch, tok.data_ptr(),
                         par.data_ptr(), cu.data_ptr(), au.data_ptr(), su.data_ptr(), B, T, V, W, path.data_ptr(),
                         num_accepted.data_ptr(), next_token.data_ptr(), ws.data_ptr(), cur)
    if st:
        if st == _native.DSA_ERR_OVERLAP:
            _fail("path, num_accepted and next_token must share memory neither with each other nor with the inputs")
        _native.check(st, "dsa_verify_run")
    if _CHECK and not torch.cuda.is_current_stream_capturing():
        raise_on_device_status(dev)


def device_status(device: torch.device, clear: bool = True) -> int:
    """OR of the sticky status bits of every workspace of this operator on
    `device` (synchronises)."""
    return read_status(device, "verify", clear)


def raise_on_device_status(device: torch.device) -> None:
    bits = device_status(device, clear=True)
    if bits:
        raise _native.DsaError(f"dsa_verify: {_native.describe_device_status(bits)} (status bits {bits:#x})")
