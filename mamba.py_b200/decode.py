"""Decoding many requests at once: their states in slots of pools, prompts read end to end, beams searched on the slots.

The reference keeps one cache per batch, in which row b belongs to request b (`Mamba.step`, mambapy/mamba.py:87).  Here a request owns a slot,
so that requests come and go, and beams go on from one another, without gathering and scattering states.
"""
from __future__ import annotations

import torch

from . import mamba as _m
from .beam import beam_reorder, beam_select


class StatePool:
    """The states and convolution windows of `slots` requests for every layer of a stack (an object with `layers` whose mixers have the
    attributes of the reference's MambaBlock).  `dtype` is the activations': the windows have it, states are float32.  Tokens and beams go
    with any d_conv up to 8, prompts with 4 alone."""

    def __init__(self, stack, slots, dtype=torch.float32, device="cuda"):
        self.stack = stack
        self.caches = []
        for layer in stack.layers:
            W, N = layer.mixer.A_log.shape
            K = layer.mixer.conv1d.weight.shape[-1]
            self.caches.append((torch.zeros(slots, W, N, dtype=torch.float32, device=device),
                                torch.zeros(slots, W, K - 1, dtype=dtype, device=device)))

    def pools(self):
        return [t for cache in self.caches for t in cache]

    @torch.no_grad()
    def prompts(self, x, cu_seqlens, slots, resume=None, max_length=None):
        """x (T, D): the embedded tokens of requests laid end to end.  Returns the stack's output for every token."""
        return _m.stack_packed(self.stack, x, cu_seqlens, self.caches, slots, resume, max_length)

    @torch.no_grad()
    def step(self, x, slots):
        """x (B, D): one embedded token a request."""
        return _m.stack_slot_step(self.stack, x, self.caches, slots)

    def reorder(self, slots, parents):
        return beam_reorder(slots, parents, self.pools())


@torch.no_grad()
def beam_search(pool, embed, head, logits, slots, steps, end_token=None):
    """`steps` tokens of a beam search.  slots (G, K), all different: slots[:, 0] has read a group's prompt (and whatever tokens have come
    since), the others may hold anything; `logits` (G, V) are those of the last token that slots[:, 0] has read.  embed(tokens (B,)) -> (B, D)
    and head(x (B, D)) -> (B, V) are the model's ends.  Returns (tokens (G, K, steps), scores (G, K)), best beam first; a beam that has chosen
    `end_token` goes on choosing it."""
    G, K = slots.shape
    scores = torch.full((G, K), float("-inf"), device=slots.device)
    scores[:, 0] = 0.0
    logits = logits[:, None, :].expand(-1, K, -1)          # (one beam that counts, until the first choice)
    finished = None if end_token is None else torch.zeros(G, K, dtype=torch.bool, device=slots.device)
    chosen = torch.empty(G, K, 0, dtype=torch.long, device=slots.device)
    for i in range(steps):
        scores, tokens, parents = beam_select(logits, scores, finished=finished, end_token=end_token)
        chosen = torch.cat([chosen.gather(1, parents[..., None].expand(-1, -1, i)), tokens[..., None]], 2)
        if finished is not None:
            finished = finished.gather(1, parents) | (tokens == end_token)
        if i + 1 < steps:
            slots = pool.reorder(slots, parents)
            logits = head(pool.step(embed(tokens.reshape(-1)), slots.reshape(-1))).view(G, K, -1)
    return chosen, scores
