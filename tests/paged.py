"""Plain forms in 64 bits of the operators over a paged cache, on the CPU, and bounds of what rounding may do to them."""
import torch

E4M3 = torch.float8_e4m3fn


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def cache_values(cache):
    """What a PagedCache stands for: k and v [pages, page, heads, dim] in fp64 on the CPU."""
    out = []
    for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = (t.float() if t.dtype == E4M3 else t).double().cpu()
        out.append(x if s is None else x * s.double().cpu()[:, None])
    return out


def attention(q, kv, tables, lengths, first, n_new, scale, window=0, max_new=None):
    """(out, bound, rows): fp64 outputs [T, Hq, D] of the requests' rows (zeros elsewhere), how far the kernel's may be from them, and
    which rows belong to a request.

    The bound: the stored output is off by half a step of itself, every weight by half a step of dtype (its sum is that of the
    unrounded ones), so their product by half a step of sum p |v|. A score is a sum of D products in fp32, each order of which is
    off by at most D 2^-24 of the sum of absolute products, A; with its factor and the exponential's argument (a few more
    roundings of at most A) that is (D + 8) 2^-24 A, and the same for the row's maximum: a weight and the sum are off by twice that of
    themselves each. Sums over the keys and the joins of pieces add at most 2^-18 of them."""
    k, v = kv
    T, hq, D = q.shape
    page, hkv = k.shape[1], k.shape[2]
    group, u = hq // hkv, half_step(q.dtype)
    x = q.double().cpu()
    out, bound = torch.zeros((T, hq, D), dtype=torch.float64), torch.zeros((T, hq, D), dtype=torch.float64)
    rows = torch.zeros((T,), dtype=torch.bool)
    tables = tables.cpu()
    for b in range(tables.shape[0]):
        n, f, length = int(n_new[b]), int(first[b]), int(lengths[b])
        if n < 0 or (max_new is not None and n > max_new) or f < 0 or f + n > T:
            continue
        rows[f:f + n] = True
        top = min(max(length, 0), tables.shape[1] * page)
        j = torch.arange(top)
        ids = tables[b].long()[j // page]
        ok = (ids >= 0) & (ids < k.shape[0])
        kk, vv = k[ids.clamp(0, k.shape[0] - 1), j % page], v[ids.clamp(0, k.shape[0] - 1), j % page]
        for i in range(n):
            p = max(length, 0) - n + i
            see = ok & (j <= p)
            if window:
                see &= j > p - window
            at = see.nonzero()[:, 0]
            if not len(at):
                continue
            for h in range(hq):
                ks, vs = kk[at, h // group], vv[at, h // group]
                s = (ks @ x[f + i, h]) * scale
                w = torch.softmax(s, 0)
                out[f + i, h] = w @ vs
                a = float((ks.abs() @ x[f + i, h].abs()).max()) * scale
                bound[f + i, h] = u * out[f + i, h].abs() + (u + 4 * (D + 8) * 2.0 ** -24 * a + 2.0 ** -18) * (w @ vs.abs())
    return out, bound * 1.01 + torch.finfo(q.dtype).tiny, rows


def turned(x, weight, positions, rotary, eps):
    """Rows [T, H, D] normed and turned, in fp64."""
    x = x.double().cpu()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double().cpu()
    if rotary is None or not rotary.inv_freq.numel():
        return x
    f = rotary.inv_freq.cpu()
    half = f.numel()
    pos = positions.cpu().double()
    pos = pos[None] if pos.dim() == 1 else pos
    axes = torch.zeros((half,), dtype=torch.long) if rotary.axes is None else rotary.axes.cpu().long()
    t = (pos[axes].t() * f)[:, None]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rotary.adjacent else (slice(0, half), slice(half, 2 * half))
    y = x.clone()
    y[..., a] = (x[..., a] * t.cos() - x[..., b] * t.sin()) * rotary.scale
    y[..., b] = (x[..., b] * t.cos() + x[..., a] * t.sin()) * rotary.scale
    return y


def turned_bound(x, weight, want, dtype, rotary=None, eps=1e-6):
    """How far a turned row of fp32 arithmetic, rounded to dtype once, may be from `want`: half a step of itself, and 2^-20 of the
    larger of its pair (some twenty roundings of 2^-24 on the way: squares summed in 8 + 5 steps, the root, two products, the angle's
    sine and cosine, two products and their sum), which the row's largest element bounds."""
    big = want.abs().amax(-1, keepdim=True)
    return (half_step(dtype) * want.abs() + 2.0 ** -19 * big) * 1.001 + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2


def e4m3_bound(want, scale, slack):
    """The same for values kept in eight bits over `scale` [heads]: half a step of theirs (2^-4 of a normal one, 2^-10 below 2^-6),
    of a value that is off by `slack` itself."""
    s = scale.double().cpu()[:, None]
    return torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10) * 1.001 + slack * 1.07
