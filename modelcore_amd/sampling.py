"""On-device next-token sampling with a counter-based random stream per row.

``PhiloxSampler`` draws one token per row from softmax(logits / temperature) with the HIP kernel
``mcamd_sample_tokens`` (Gumbel-max with Philox4x32-10 noise; C ABI in include/modelcore_amd.h).
Row r is keyed by its own 64-bit seed (``base_seed + r`` by default) and a device-side counter
that each call advances, so:

* a row's tokens depend only on its seed, its logits and how many tokens it has drawn -- not on
  the batch it is decoded in, nor on the other rows;
* nothing is read back to the host, so a decode step that samples stays asynchronous.

This is the sampling half of modelcore/generate.py:18-34 (``sample_next_token`` with
temperature > 0, with or without top_k) restated for the device; the reference draws from one
torch.Generator for the whole batch, which has no per-row meaning. Temperature 0 is the argmax,
as in the reference. With top_k the draw is over the k largest logits of each row (ties at the
k-th value kept lowest index first).

``verify_drafts`` is the draw of a step that runs several drafted tokens a row: how many of them the
target's own distribution accepts, and the token after the last of those.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from modelcore_amd import _ext

__all__ = ["PhiloxSampler", "Verified", "verify_drafts"]


class PhiloxSampler:
    def __init__(self, batch_size, device, base_seed=0, seeds=None):
        if seeds is None:
            seeds = [base_seed + r for r in range(batch_size)]
        if len(seeds) != batch_size:
            raise ValueError(f"need {batch_size} seeds, got {len(seeds)}")
        _ext.require_rocm(torch.empty(0, device=device), what="PhiloxSampler")
        self.batch_size = batch_size
        self.seeds = torch.tensor([s & (2 ** 64 - 1) for s in seeds], dtype=torch.uint64,
                                  device=device)
        self.offsets = torch.zeros(batch_size, dtype=torch.int64, device=device)

    def __call__(self, logits, temperature=1.0, top_k=None):
        """(B, V) logits -> (B, 1) int64 token ids; advances every row's counter by one."""
        _ext.require_rocm(logits, what="PhiloxSampler")
        if logits.dim() != 2 or logits.size(0) != self.batch_size:
            raise ValueError(f"logits must be ({self.batch_size}, vocab); got {tuple(logits.shape)}")
        if temperature < 0:
            raise ValueError("temperature must be non-negative")
        if logits.dtype != torch.float32:
            logits = logits.float()
        if logits.stride(1) != 1 or 0 < logits.stride(0) < logits.size(1):
            logits = logits.contiguous()  # a stride-0 (expanded) batch is read as is
        out = torch.empty(self.batch_size, dtype=torch.int64, device=logits.device)
        st = _ext.lib().mcamd_sample_tokens(
            logits.data_ptr(), self.batch_size, logits.size(1), logits.stride(0),
            float(temperature), int(top_k or 0), self.seeds.data_ptr(), self.offsets.data_ptr(),
            out.data_ptr(),
            _ext.stream_handle(logits.device))
        _ext.check(st, "sample_tokens")
        return out.view(-1, 1)


class Verified(NamedTuple):
    """How far each row's drafts go (``verify_drafts``)."""
    kept: torch.Tensor    # (rows, max_seqlen) int32: the accepted nodes, the root first, then -1
    counts: torch.Tensor  # (rows,) int32: how many (0 for a row without nodes)
    tokens: torch.Tensor  # (rows, max_seqlen) int64: the tokens after the root, as many, then -1


@functools.lru_cache(maxsize=1024)
def _verify_scratch_bytes(total, vocab):
    return _ext.lib().mcamd_verify_drafts_scratch_bytes(total, vocab)


def verify_drafts(logits, tokens, parents, cu_seqlens, numbers, *, temperature=1.0, draft_probs=None,
                  max_seqlen) -> Verified:
    """Walks each row's drafted tree from its root as far as the target's logits accept, and draws the token
    after the last accepted node; tokens so emitted are a draw from softmax(logits / temperature), token by
    token, whatever the drafts were.

    Args:
        logits: (total, vocab), the target's at every node, the rows' nodes one after another (fp32; others
            are converted)
        tokens: (total,) int64, the nodes' tokens; node 0 of a row, its root, is the token it ended with
        parents: (total,) int32, as ``paged_tree``
        cu_seqlens: (rows + 1,) int32 offsets of the rows
        numbers: (total,) fp32 random numbers from [0, 1), one a node; the root's is the draw's
        temperature: of the softmax; 0 takes the largest logits (the first of equal ones)
        draft_probs: (total, vocab) fp32, row i the distribution that the children of node i were drawn
            from, independently of one another (rows of nodes without children are not read); None where
            the drafts are guesses; a vocabulary of at most 2^23 tokens then
        max_seqlen: at least the nodes of the widest row (host int), at most 1024; a row's nodes past it
            are left out

    At a node the children are tried in the order of their indices. Drawn from q, x is accepted if number * Z *
    q(x) < max(p(x) - a q(x), 0), where a = 0 and Z = 1, and after each that is refused a + Z and sum(max(p -
    a q, 0)). A guess is accepted if number * Z < p(x), Z being 1 less the p of those refused before it. The
    last token is drawn from what is left of p. Probabilities are in 64 bits; one up to 1e-290 of the largest is 0.
    -inf and NaN logits are probability 0 (so a caller's top_k is a mask of -inf, or of the type's lowest value); of
    a node with no others nothing is accepted and the last token is 0. A child whose token is outside the
    vocabulary is passed over.
    """
    what = "verify_drafts"
    _ext.require_rocm(logits, what=what)
    dev = logits.device
    _ext.same_device(dev, tokens=tokens, parents=parents, cu_seqlens=cu_seqlens, numbers=numbers,
                     draft_probs=draft_probs)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be (total, vocab); got {tuple(logits.shape)}")
    total, vocab = logits.shape
    for name, t, dtype in (("tokens", tokens, torch.int64), ("parents", parents, torch.int32),
                           ("numbers", numbers, torch.float32)):
        if t.dtype != dtype or t.shape != (total,):
            raise ValueError(f"{name} must be ({total},) {dtype}; got {tuple(t.shape)} {t.dtype}")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be (rows + 1,) int32")
    if temperature < 0:
        raise ValueError("temperature must be non-negative")
    max_seqlen = int(max_seqlen)
    if not 1 <= max_seqlen <= 1024:
        raise ValueError(f"max_seqlen must be 1 to 1024; got {max_seqlen}")
    if draft_probs is not None and (draft_probs.shape != logits.shape or draft_probs.dtype != torch.float32):
        raise ValueError(f"draft_probs must be {tuple(logits.shape)} fp32; got {tuple(draft_probs.shape)} "
                         f"{draft_probs.dtype}")

    def rows_of(t):
        return t if t.stride(1) == 1 and (t.stride(0) >= vocab or total <= 1) or vocab == 1 and total <= 1 \
            else t.contiguous()

    logits = rows_of(logits.float())
    probs = None if draft_probs is None else rows_of(draft_probs)
    tokens, parents, numbers, cu_seqlens = (t.contiguous() for t in (tokens, parents, numbers, cu_seqlens))
    n = cu_seqlens.numel() - 1
    kept = parents.new_empty((n, max_seqlen))
    counts = parents.new_empty((n,))
    out = tokens.new_empty((n, max_seqlen))
    with _ext.on_device(dev):
        nbytes = _verify_scratch_bytes(total, vocab)
        # Scratch of the call's own: calls on several streams, and captured graphs, share nothing.
        ws = logits.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        st = _ext.lib().mcamd_verify_drafts(
            logits.data_ptr(), max(logits.stride(0), vocab), probs.data_ptr() if probs is not None else None,
            max(probs.stride(0), vocab) if probs is not None else 0, tokens.data_ptr(), parents.data_ptr(),
            cu_seqlens.data_ptr(), numbers.data_ptr(), kept.data_ptr(), counts.data_ptr(), out.data_ptr(),
            n, total, max_seqlen, vocab, float(temperature), ws.data_ptr() if ws is not None else None,
            nbytes, _ext.stream_handle(dev))
    _ext.check(st, what)
    return Verified(kept, counts, out)
