"""Token sampling: temperature, top-k, top-p and min-p from given uniform
numbers.

The reference's harness (bench_fused_cpm5.py:27-57) takes the most likely token
of every step (llama.greedy here).  The definition, with its ties and empty
rows, is in include/bf16x_llama.h; the kernels are csrc/sample.hip.
"""
from __future__ import annotations

from . import _lib

__all__ = ["sample"]


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, token=None, state=None, history=None):
    """(token int64 [rows], logprob fp32 [rows]) drawn from logits [rows, vocab]
    (or [vocab]; bf16, fp16 or fp32, rows may be strided) with the uniform
    numbers u (fp32 [rows], in [0, 1)).

    temperature, top_k, top_p, min_p: numbers, or tensors of one per row (top_k
    int32, the others fp32).  The filters apply in this order: top_k tokens,
    the fewest of them with top_p of their weight, those of at least min_p of the
    likeliest one's weight; top_k 0, top_p 1, min_p 0 keep everything, and
    temperature 0 takes the maximum.  logprob is the token's among those kept.
    Equal logits are kept lowest index first.  A row of only -inf or NaN gives
    token -1.

    token: the int64 tensor to write to.  state (int32 [2], one row): the step's
    number is u[state[1]], history[state[1]] gets the token, and both counts of
    state go up by one, as llama.greedy does, so that a captured decode step
    draws a new number every time it is replayed."""
    r = _lib.host().sample(logits, u, temperature, top_k, top_p, min_p, token, state, history)
    if isinstance(r, int):
        _lib.check(r, "bf16x_sample")
    return r
