"""Trees of drafted tokens: what a parent list means for masks and positions.

A tree over T drafted tokens is given by each token's parent, an index below
its own, or a negative number for a token that continues the cached context
itself.  ``BatchedPagedKVCache.attend_tree`` takes the visibility mask that
follows from it; the rotary position of a token is its sequence's cached
length plus its depth.
"""
from __future__ import annotations

import torch


def tree_mask(parents) -> torch.Tensor:
    """Bool mask [..., T, T] of a parent list or tensor [..., T]: True where
    token t sees token u, that is u is t or one of its ancestors.  A parent that is not
    below its token is refused (on the device, where looking would wait: counts as none)."""
    p = torch.as_tensor(parents).long()
    T = p.shape[-1]
    i = torch.arange(T, device=p.device)
    if p.device.type == "cpu" and bool((p >= i).any()):
        raise ValueError("a token's parent must have a smaller index than the token")
    p = torch.where(p < i, p, -1)
    # seen: ancestors at distances below reach; up: the ancestor at distance reach
    seen = (i[:, None] == i).expand(*p.shape, T)
    up, reach = p, 1
    while reach < T:
        at = up.clamp(min=0)[..., None].expand(*up.shape, T)
        seen = seen | (seen.gather(-2, at) & (up >= 0)[..., None])
        up = torch.where(up >= 0, up.gather(-1, up.clamp(min=0)), up)
        reach *= 2
    return seen


def tree_depths(mask: torch.Tensor) -> torch.Tensor:
    """Depth of every token of a tree mask [..., T, T]: its ancestors' count."""
    return mask.sum(-1) - 1
