"""Beam search over sequences whose states lie in slots of pools: the two operations between one decode step and the next.

The reference samples; it has no counterpart.  Both run on the device without a synchronisation, so that a whole step of a search
(layers on slots, `beam_select`, `beam_reorder`) can be captured into a graph.
"""
from __future__ import annotations

from ._lib import host as _host


def beam_select(logits, scores, num=None, finished=None, end_token=None):
    """The best continuations of each group's beams, over beams and vocabulary.

    logits : (G, K, V) or (G * K, V), float32 or bfloat16   scores : (G, K) float32, the beams' log-probabilities so far.
    Returns (scores (G, num) float32, tokens (G, num), parents (G, num)), highest first: a continuation's score is its beam's plus the
    token's log-softmax; equal ones come in the order of parent and token.  `num` is K by default; 2 K lets a caller put ended ones aside.
    A beam that `finished` (G, K) bool marks has one continuation, `end_token`, at its own score.  A beam whose score is not finite (the
    others of a search's first step: -inf) or whose logits hold a NaN, +inf or nothing above -inf has none.  Places left are filled with
    the lowest tokens of the lowest beams at -inf.  K and num are at most 64, G * K at most 65535."""
    return _host().beam_select(logits, scores, num, finished, end_token)


def beam_reorder(slots, parents, pools):
    """The slots of the beams that go on, and the copies this takes, in all `pools` at once.

    slots, parents : (G, K); parents[g, i] is the beam of group g that beam i goes on from (what `beam_select` returns, narrowed to K).
    pools : tensors of one number of slots each (states and windows of every layer), updated in place.  Returns the new slots (G, K): the
    lowest child of a beam keeps its slot; the other children take the slots of beams without children, lowest first, and only their
    entries are copied.  A parent that is no beam is nobody: its child gets a slot with what is in it.  Slots must differ; those outside
    the pools are handed on, and nothing is copied to or from them.  At most 64 beams a group and 4096 in a call."""
    return _host().beam_reorder(slots, parents, pools)
