"""Log-probabilities of given tokens under rows of logits, with their ranks, the rows' entropies and the likeliest alternatives
(esp_token_logprobs, csrc/logprobs.hip): what follows the LM head when a request asks for them, or a prompt is scored.
"""
from __future__ import annotations

from .experts import ext


def token_logprobs(logits, tokens, top: int = 0, temperature=None, out=None):
    """(logprobs fp32 [R], ranks int32 [R], entropies fp32 [R], top_ids int32 [R, top], top_logprobs fp32 [R, top]).

    logits       [R, V], bf16, fp16 or fp32, rows that start at any element, V at most 2^20. Masked tokens are -inf.
    tokens       int32 [R]; one outside [0, V): rank and log-probability 0
    top          how many of the likeliest tokens, at most 64; among equal ones the lowest first
    temperature  fp32 [R]: p = softmax(row / temperature); below 1e-5 (a greedy request), or None: 1
    out          the five to write into, apart from one another and from the inputs; otherwise new ones

    A rank is 1 + the number of tokens with a larger logit, or an equal one and a lower index. A row without a distribution (a NaN
    or +inf in it, or nothing above -inf) has NaN for its entropy and its log-probabilities. A row's bits depend on that row alone;
    nothing is kept between calls, so calls on several streams do not meet."""
    return ext().token_logprobs(logits, tokens, top, temperature, out)
