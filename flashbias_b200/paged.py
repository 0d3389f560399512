"""Serving over a paged cache: the plan of a step, the append of its tokens, and attention with the framework's biases.

A cache is a pool of pages, ``(num_pages, page_size, nheads_k, headdim)`` each for keys and values (any page, place and head
strides), and with low-rank factors a third of their key side, ``(num_pages, page_size, nheads_k | 1, rank)``.  A step is

    plan = paged_plan(block_table, pages_held, free_pages, free_count, lens, new_lens, page_size, num_tokens, parents)
    q = paged_append(q, k, v, key_cache, value_cache, plan.slots, plan.positions, inv_freq, ...)          # per layer
    o = flash_bias_paged_func(q, key_cache, value_cache, block_table, plan.lens, plan.cu_tokens,          # per layer
                              plan.tree_mask, plan.positions, slopes=slopes)

with everything on the device and nothing read back, so that a step can be captured in a CUDA graph.  The reference has no
cache: its operator takes dense tensors (flash_bias/flash_bias_triton.py:1345-1405).  Inference only.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch

from .flash_bias import _op

__all__ = ["PagedPlan", "paged_plan", "paged_append", "flash_bias_paged_func"]


class PagedPlan(NamedTuple):
    """What ``paged_plan`` found out, on the device."""
    slots: torch.Tensor  # (num_tokens) int64: place of each new token in the cache, -1 for none
    positions: torch.Tensor  # (num_tokens) int32
    cu_tokens: torch.Tensor  # (requests + 1) int32: first new token of each request
    lens: torch.Tensor  # (requests) int32: cached tokens in front of the new ones, -1 for a refused request
    tree_mask: Optional[torch.Tensor]  # (num_tokens, words) int64: the ancestors of each token as bits


def paged_plan(block_table: torch.Tensor, pages_held: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
               lens: torch.Tensor, new_lens: torch.Tensor, page_size: int, num_tokens: int,
               parents: Optional[torch.Tensor] = None, max_tree: int = 64) -> PagedPlan:
    """Fit the pages of every request to ``lens + new_lens`` tokens, and place the new tokens.

    block_table (requests, width), pages_held (requests), free_pages (pool, a stack) and free_count (1): int32, the state of
        the pool, updated in place.  Pages that a request no longer needs go back to the stack (``lens = new_lens = 0`` frees
        a request), missing ones are taken from its top, in the order of the requests.  Counts that do not fit the table
        or the stack are reported as device-side errors.
    lens, new_lens: (requests) int32.  num_tokens: rows of the step's token tensors; what the requests do not fill is padding.
    parents: (num_tokens) int32, for trees of drafted tokens: index within its request of each token's parent, which comes
        before it; negative for the cached context.  None: each token follows the one before.
    max_tree: most drafted tokens of a request (the words of ``tree_mask`` are made for it).

    A request is refused (``lens`` -1, its tokens without slots, its pages as they were) when the free pages do not last, its
    row of the table is too short, its tokens pass ``num_tokens``, its tree has more than ``max_tree`` tokens (rounded up to 64)
    or a length is negative; the others are served.
    """
    return PagedPlan(*_op().paged_plan(block_table, pages_held, free_pages, free_count, lens, new_lens, page_size, num_tokens,
                                       parents, max_tree))


def paged_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                 slots: torch.Tensor, positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 axes: Optional[Sequence[int]] = None, interleaved: bool = False, eps: float = 1e-6,
                 k_bias: Optional[torch.Tensor] = None, bias_cache: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """``norm_rope_func`` on flat tokens, with the keys, the values and the keys' bias factors written to their slots.

    q: (tokens, nheads, headdim) or None; k, v: (tokens, nheads_k, headdim); k_bias: (tokens, nheads_k | 1, rank).
    slots: (tokens) int32 or int64, ``page * page_size + place``; negative: the token is padding and nothing is written.  A slot
        behind the cache is not written either and reported as a device-side error.  No slot may occur twice in a call, and
        what is appended may not lie in a cache itself, nor may two caches share elements.
    positions: (tokens), or with axes (A, tokens).  The other arguments are those of ``norm_rope_func``; without positions and
        weights the keys are stored as they are.

    Returns the normalised and rotated q as a new tensor (None without q).
    """
    return _op().paged_append(q, k, v, key_cache, value_cache, slots, positions, inv_freq, q_weight, k_weight, axes, interleaved,
                              eps, k_bias, bias_cache)


def flash_bias_paged_func(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                          lens: torch.Tensor, cu_tokens: torch.Tensor, tree_mask: Optional[torch.Tensor] = None,
                          positions: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None,
                          q_bias: Optional[torch.Tensor] = None, bias_cache: Optional[torch.Tensor] = None,
                          softmax_scale: Optional[float] = None, return_lse: bool = False):
    """Attention of every request's newest tokens over its pages, their own keys among them.

    q: (tokens, nheads, headdim), nheads a multiple of the cache's heads; request b owns tokens ``cu_tokens[b]`` to
        ``cu_tokens[b + 1]`` and its keys are the first ``lens[b]`` places of its pages and one for each of those tokens.
    tree_mask: (tokens, words) int64; bit j % 64 of word j / 64 lets a token see the request's j-th new token.  None: a token
        sees the new ones up to itself.  The cached keys are seen by all.
    slopes: (nheads): adds ``slope * (key position - token position)``, where a cached key's position is its place and a new
        token's is ``positions`` (int32; None: its place).  Positions may lie anywhere; differences up to 2^24 between the tokens
        of a request are exact.
    q_bias (tokens, nheads | 1, rank) with bias_cache: adds ``q_bias . k_bias``.  Not together with slopes.
    softmax_scale: multiplies q.k only; None or 0: 1 / sqrt(headdim).

    Returns o (tokens, nheads, headdim), with ``return_lse`` also the fp32 log-sum-exp (tokens, nheads).  Rows that see no key,
    tokens of a refused request (``lens`` -1) and tokens of no request yield 0 / -inf.  A bias may be as low as the type allows: a
    row whose keys all carry it is what its logits say, and only a logit of -inf counts as a key that is not seen.
    """
    o, lse = _op().paged_forward(q, key_cache, value_cache, block_table, lens, cu_tokens, tree_mask, positions, slopes, q_bias,
                                 bias_cache, softmax_scale, return_lse, 0)
    return (o, lse) if return_lse else o
