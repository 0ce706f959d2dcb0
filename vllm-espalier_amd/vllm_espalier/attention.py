"""What stands between a layer's q/k/v projections and its output projection when it serves requests: the new tokens' keys and
values into a paged cache, with the norms and the rotation of queries and keys on the way (esp_cache_append, csrc/cache.hip), and
the attention of the new tokens over that cache (esp_paged_attention, csrc/attention.hip).

A cache's memory belongs to no request: it is pages of a fixed number of tokens, and every request has a table of the pages that
are its own, in order. What a captured graph holds are the addresses of the cache, the tables and the lengths, whose contents may
change from replay to replay.
"""
from __future__ import annotations

import torch

from .experts import ext

DIMS = (64, 128, 256)        # elements of a head
PAGE_UNIT = 16               # a page's tokens are a multiple of this
PIECE_UNIT = 128             # and so are a piece's of this (attend's split)


class Rotary:
    """The rotation of positions: pair f of a head's first 2 * len(inv_freq) elements turns by position * inv_freq[f].

    inv_freq   fp64 [half]: any base and any scaling of it is a matter of these numbers; half a multiple of 8
    axes       int32 [half]: which of several positions (time, height, width) each pair turns with; None: all with the first
    adjacent   a pair is elements 2 f and 2 f + 1; otherwise f and half + f
    scale      a factor of the turned pairs"""

    def __init__(self, inv_freq: torch.Tensor, axes: torch.Tensor | None = None, adjacent: bool = False, scale: float = 1.0):
        if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64 or inv_freq.numel() % 8:
            raise ValueError("inv_freq: fp64, one number a pair, a multiple of 8 of them")
        if axes is not None and (axes.dtype != torch.int32 or axes.shape != inv_freq.shape):
            raise ValueError("axes: int32, one number a pair")
        self.inv_freq = inv_freq.contiguous()
        self.axes = None if axes is None else axes.contiguous()
        self.adjacent, self.scale = bool(adjacent), float(scale)

    @classmethod
    def of_base(cls, elements: int, base: float = 10000.0, sections=None, interleaved: bool = False, device="cuda", **more):
        """base^(-2 f / elements) for the pairs of `elements` elements. sections: how many pairs each axis has, one axis after
        the other, or (interleaved) in turn, pair f on axis f mod the number of axes as long as that one has pairs left, else on
        axis 0. An axis behind the first that has more pairs than turns is refused."""
        half = elements // 2
        if elements <= 0 or elements % 16:
            raise ValueError("a rotation takes a positive multiple of 16 elements")
        inv_freq = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
        axes = None
        if sections is not None:
            sections = [int(n) for n in sections]
            if any(n < 0 for n in sections) or sum(sections) != half:
                raise ValueError(f"sections: numbers of pairs that add up to {half}")
            if interleaved:
                left, order = list(sections), []
                for f in range(half):
                    a = f % len(sections)
                    order.append(a if f // len(sections) < left[a] else 0)
                if [order.count(a) for a in range(len(sections))] != sections:
                    raise ValueError(f"sections: an axis has more pairs than turns among {half} interleaved ones")
            else:
                order = [a for a, n in enumerate(sections) for _ in range(n)]
            axes = torch.tensor(order, dtype=torch.int32, device=device)
        return cls(inv_freq.to(device), axes, **more)


class PagedCache:
    """The keys and values of a layer in pages: k and v [pages, page, heads, dim] of any strides with a head's elements side by
    side (16-byte aligned), bf16, fp16 or e4m3. e4m3 has a scale a head (fp32 [heads], positive) for k and for v: a value stands
    for itself times its head's scale. dim is 64, 128 or 256, page a multiple of 16. append needs k and v apart; attend may have one
    tensor for both."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v: [pages, page, heads, dim] of one dtype")
        if k.dtype not in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
            raise ValueError("a cache is bf16, fp16 or e4m3")
        if k.shape[3] not in DIMS or k.shape[1] % PAGE_UNIT or 0 in k.shape:
            raise ValueError(f"heads of {DIMS} elements, pages of a multiple of {PAGE_UNIT} tokens")
        for scale in (k_scale, v_scale):
            if (scale is not None) != (k.dtype == torch.float8_e4m3fn):
                raise ValueError("an e4m3 cache has a scale a head for k and for v, one of 16 bits has none")
            if scale is not None and (scale.dtype != torch.float32 or scale.shape != k.shape[2:3]):
                raise ValueError("scales: fp32, one a head")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages: int, page: int, heads: int, dim: int, dtype=torch.bfloat16, device="cuda", k_scale=None, v_scale=None):
        """A cache of zeros, a page's tokens of one head side by side. e4m3 scales: a number, or one a head."""
        k, v = (torch.zeros((pages, heads, page, dim), dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
        scales = [None if s is None else torch.as_tensor(s, dtype=torch.float32, device=device).expand(heads).contiguous()
                  for s in (k_scale, v_scale)]
        return cls(k, v, *scales)

    def append(self, q, k, v, slots, positions=None, rotary: Rotary | None = None, q_norm=None, k_norm=None, eps: float = 1e-6,
               out=None):
        """The queries of T new tokens, normed and turned (`out`, or a new tensor; out may be q); their keys, normed and turned,
        and values into the cache.

        q [T, query heads, dim], k and v [T, heads, dim] (bf16 or fp16, views of one q/k/v buffer as they are), slots int64 [T]:
        page * (tokens a page) + token in the page, different ones; outside the cache (-1, the padding of a batch) nothing is
        stored. positions int64 [T], or [axes, T]. q_norm, k_norm: RMSNorm weights [dim] of q's dtype, or None.
        A row's bits depend on that row alone."""
        turn = (None, None, False, 1.0) if rotary is None else (rotary.inv_freq, rotary.axes, rotary.adjacent, rotary.scale)
        return ext().cache_append(q, k, v, self.k, self.v, self.k_scale, self.v_scale, slots, positions, *turn, q_norm, k_norm,
                                  eps, out)

    def attend(self, q, tables, lengths, first=None, n_new=None, max_new: int = 1, scale: float | None = None, window: int = 0,
               split: int = 0, out=None):
        """The attention of B requests' new tokens over what the cache holds of each request, themselves included: [T, query
        heads, dim] (`out`, apart from q, or a new tensor).

        q         [T, query heads, dim], query heads a multiple of the cache's
        tables    int32 [B, pages a request]: token j of request b is in page tables[b, j // page]; an entry outside the cache
                  hides its tokens
        lengths   int32 [B]: a request's tokens in the cache, its new ones the last of them
        first, n_new  int32 [B]: its new tokens are rows first .. first + n_new of q, its own (default, with max_new 1: row b);
                  n_new outside [0, max_new]: no such request, the padding of a fixed batch
        max_new   the most that n_new may hold: what the launches are sized for
        scale     of the scores; default 1 / sqrt(dim)
        window    how many tokens a row sees, its own the last; 0: all
        split     tokens a piece of a request's keys (a multiple of 128) where pieces run apart; 0: chosen on the device from
                  the batch's lengths. With a split of its own a row's bits depend on its request alone (one of more than 32 rows
                  a head of the cache, n_new times the heads of a group, is then not cut: few such rows over many tokens take long).
                  Scratch and launch are then sized by what the tables could hold.

        Rows that see nothing are zeros; rows of no request are left as they are (in a new tensor: undefined). Nothing is kept
        between calls, so calls on several streams do not meet."""
        return ext().paged_attention(q, self.k, self.v, self.k_scale, self.v_scale, tables, lengths, first, n_new, max_new,
                                     self.k.shape[3] ** -0.5 if scale is None else scale, window, split, out)
