"""Verification of drafted tokens against the target's logits (esp_verify, csrc/verify.hip): what follows the LM head when the
rows of a batch are a request's last token and its drafts (an MTP drafter's or any other's).
"""
from __future__ import annotations

from .experts import ext


def verify(logits, first, n_drafts, drafts, uniform, race, temperature, draft_probs=None, out=None):
    """(tokens int32 [B, G + 1], counts int32 [B], logprobs fp32 [B, G + 1]) of B requests with up to G drafts each: the drafts
    accepted, then one token drawn from the target, then -1 (log-probabilities 0).

    logits       [R, V], bf16, fp16 or fp32: request b's rows are first[b] .. first[b] + n_drafts[b], the target's logits at
                 its drafts' positions and at the one behind them. Masked tokens are -inf.
    first, n_drafts  int32 [B]; n_drafts of -1 (or anything outside [0, G]): no such request, the padding of a fixed batch
    drafts       int32 [B, G], those past n_drafts unused
    uniform      fp32 [B, G] in [0, 1): draft j is accepted iff uniform * q(draft) < p(draft), p = softmax(row / temperature)
    race         fp32 [B, V], exponentially distributed: the token drawn is the argmax of w / race, w = max(p - q, 0) at the
                 first rejected draft, p behind the last accepted one
    temperature  fp32 [B]; below 1e-5: greedy (a draft is accepted iff it is the row's argmax)
    draft_probs  fp32 [B, G, V], what the drafts were drawn from (q); None: the drafter was sure (q = 1 at its draft)
    out          (tokens, counts, logprobs) to write into, apart from one another and from the inputs; otherwise new ones

    Acceptance is decided in 64 bits from sums of 32, the race in 32 bits: what is decided by less than about 2^-19 of p may fall on
    either side, the same one in every call with these inputs.

    With fixed arrays a captured graph replays it; nothing is kept between calls, so calls on several streams do not meet."""
    return ext().verify(logits, first, n_drafts, drafts, uniform, race, temperature, draft_probs, out)
