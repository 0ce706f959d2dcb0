"""GPU checks of the paged cache's appends and of the attention over it against plain forms in 64 bits (paged.py), at the sizes,
masks and layouts where they can go wrong. Bounds are derived there."""
import pytest
import torch

import paged
from vllm_espalier.attention import PagedCache, Rotary

pytestmark = pytest.mark.gpu
BF, HF, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make_cache(gen, dev, pages, page, heads, dim, dtype, nhd=False, fill=None):
    """A cache of normal values, in either order of tokens and heads; fill: what it holds instead."""
    shape = (pages, page, heads, dim) if nhd else (pages, heads, page, dim)
    scale = None
    if dtype == E8:
        scale = (0.02 + 0.01 * torch.arange(heads) / heads).to(dev), torch.full((heads,), 0.03, device=dev)
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen) * (30.0 if dtype == E8 else 1.0) if fill is None else torch.full(shape, fill)
        x = x.to(dtype).to(dev)
        out.append(x if nhd else x.transpose(1, 2))
    return PagedCache(*out, *(scale or ()))


def make_tables(gen, dev, held, pages, width, spare=0):
    """Tables of `width` pages in any order; entries past a request's own are `spare`."""
    order = torch.randperm(pages, generator=gen)
    t, at = torch.full((len(held), width), spare, dtype=torch.int32), 0
    for b, n in enumerate(held):
        t[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    return t.to(dev)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def compare(got, want, bound, rows=None):
    got = got.double().cpu()
    if rows is not None:
        got, want, bound = got[rows], want[rows], bound[rows]
    assert torch.isfinite(got).all()
    off = (got - want).abs() / bound
    assert float(off.max()) <= 1.0, f"{float(off.max())} of the bound at {int(off.argmax())}"


def batch(gen, dev, lengths, n_new, hq, hkv, dim, page, dtype=BF, cache_dtype=None, nhd=False, window=0, split=0, width=None, max_new=None,
          spread=1.5):
    held = [-(-max(v, 0) // page) for v in lengths]
    pages = sum(held) + 2
    cache = make_cache(gen, dev, pages, page, hkv, dim, cache_dtype or dtype, nhd)
    tables = make_tables(gen, dev, held, pages, width or max(1, max(held)))
    rows = [max(n, 0) for n in n_new]
    first = [sum(rows[:b]) for b in range(len(rows))]
    T = sum(rows) + 2
    q = (torch.randn((T, hq, dim), generator=gen) * spread).to(dtype).to(dev)
    out = torch.full((T, hq, dim), 7.0, dtype=dtype, device=dev)
    top = max_new or max(1, max(n_new))
    got = cache.attend(q, tables, i32(lengths, dev), i32(first, dev), i32(n_new, dev), top, window=window, split=split, out=out)
    assert got is out
    want, bound, mine = paged.attention(q, paged.cache_values(cache), tables, lengths, first, n_new, dim ** -0.5, window, top)
    compare(got, want, bound, mine)
    assert (out[~mine.to(dev)] == 7.0).all()                  # rows of no request stay as they are
    return cache, q, tables, first, out


@pytest.mark.parametrize("dim,hq,hkv", [(128, 32, 4), (64, 8, 8), (256, 16, 2), (128, 6, 1), (64, 64, 1), (256, 3, 3), (128, 20, 4)])
@pytest.mark.parametrize("dtype,cache_dtype", [(BF, BF), (HF, HF), (BF, E8), (HF, E8)])
def test_tokens(dev, dim, hq, hkv, dtype, cache_dtype):
    """One token a request: lengths from one to several pieces, at and beside the borders of steps, pages and pieces."""
    gen = torch.Generator().manual_seed(dim + hq)
    batch(gen, dev, [1, 2, 16, 31, 32, 33, 127, 128, 129, 200, 517], [1] * 11, hq, hkv, dim, 16, dtype, cache_dtype)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 144, 544, 65536])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pages(dev, page, dim):
    """Pages that end inside a step or a piece, and one that is longer than everything."""
    gen = torch.Generator().manual_seed(page)
    batch(gen, dev, [page + 1 if page < 1000 else 700, 333, 95, 96, 97, 1200], [1, 2, 1, 3, 1, 1], 4, 2, dim, page)


@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 128), (8, 1, 64), (4, 2, 256)])
@pytest.mark.parametrize("n_new", [[2, 1, 4, 3], [8, 5, 1, 7], [17, 16, 33, 2], [150, 1, 64, 129]])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100])
def test_drafts_and_prompts(dev, hq, hkv, dim, n_new, window):
    gen = torch.Generator().manual_seed(window + sum(n_new))
    far = [0, 40, 131, 300]
    batch(gen, dev, [n + f for n, f in zip(n_new, far)], n_new, hq, hkv, dim, 32, window=window)


@pytest.mark.parametrize("dtype,cache_dtype", [(HF, HF), (BF, E8), (HF, E8)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_of_other_types(dev, dtype, cache_dtype, dim):
    gen = torch.Generator().manual_seed(3)
    batch(gen, dev, [200, 77, 140], [190, 77, 3], 8, 2, dim, 48, dtype, cache_dtype)


def test_rows_that_see_nothing(dev):
    """Lengths below the new tokens' number, of zero and below, no request at all, too many new tokens, rows outside the batch."""
    gen = torch.Generator().manual_seed(1)
    for lengths, n_new, top in (([0, 1, 3, -5, 20, 9], [2, 3, 3, 1, 0, -1], 3), ([0], [1], 1), ([0, 40], [40, 60], 60),
                                ([30, 31], [2, 5], 4)):
        batch(gen, dev, lengths, n_new, 8, 2, 128, 16, max_new=top)
    cache = make_cache(gen, dev, 4, 16, 2, 64, BF)
    q = torch.randn((3, 4, 64), generator=gen).to(BF).to(dev)
    out = torch.full_like(q, 3.0)
    cache.attend(q, i32([[0], [1], [2]], dev), i32([5, 5, 5], dev), i32([2, -1, 3], dev), i32([2, 1, 1], dev), 2, out=out)
    assert (out == 3.0).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cache_dtype", [BF, E8])
@pytest.mark.parametrize("n_new", [1, 4, 70])
def test_hidden_places_do_not_matter(dev, dim, cache_dtype, n_new):
    """NaN wherever no request's token stands, in pages of nobody and behind the ends of pages; a page that is not there and ones
    outside the cache hide their tokens; what a window hides is NaN too."""
    gen = torch.Generator().manual_seed(n_new)
    page, hkv, lengths = 16, 2, [n_new + 5, n_new + 100, n_new + 150]
    held = [-(-v // page) for v in lengths]
    pages = sum(held) + 3
    clean = make_cache(gen, dev, pages, page, hkv, dim, cache_dtype)
    dirty = make_cache(gen, dev, pages, page, hkv, dim, cache_dtype, fill=float("nan"))
    tables = make_tables(gen, dev, held, pages, max(held) + 2, spare=pages - 1)
    for b, v in enumerate(lengths):
        j = torch.arange(v, device=dev)
        at = (tables[b].long()[j // page], j % page)
        for d, c in ((dirty.k, clean.k), (dirty.v, clean.v)):
            d.view(torch.uint8 if cache_dtype == E8 else BF)[at] = c.view(torch.uint8 if cache_dtype == E8 else BF)[at]
    tables[1, 2], tables[2, 0], tables[2, 3] = -1, pages, 2 ** 31 - 1
    q = torch.randn((3 * n_new, 8, dim), generator=gen).to(BF).to(dev)
    first = [0, n_new, 2 * n_new]
    for window in (0, 37):
        args = (q, tables, i32(lengths, dev), i32(first, dev), i32([n_new] * 3, dev), n_new)
        got = dirty.attend(*args, window=window)
        want, bound, _ = paged.attention(q, paged.cache_values(clean), tables, lengths, first, [n_new] * 3, dim ** -0.5, window)
        compare(got, want, bound)
    j = torch.arange(30, device=dev)                          # what no row of the window sees any more
    bits = torch.uint8 if cache_dtype == E8 else BF
    for d in (dirty.k, dirty.v):
        d.view(bits)[tables[1].long()[j // page], j % page] = torch.full((), float("nan")).to(cache_dtype).view(bits).to(dev)
    assert torch.isfinite(dirty.attend(*args, window=37).float()).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_token_reaches_those_that_see_it(dev, dtype, dim, hq, bad):
    """A value of a draft that is no number: the rows before it are as without it, the ones that see it are not finite; and the same for a
    key."""
    gen = torch.Generator().manual_seed(5)
    cache = make_cache(gen, dev, 8, 32, 2, dim, dtype)
    tables, length, n = i32([[3, 1, 5]], dev), 75, 6
    q = torch.randn((n, hq, dim), generator=gen).to(dtype).to(dev)
    args = (q, tables, i32([length], dev), i32([0], dev), i32([n], dev), n)
    want, bound, _ = paged.attention(q, paged.cache_values(cache), tables, [length], [0], [n], dim ** -0.5)
    page, at = (length - n + 3) // 32, (length - n + 3) % 32
    keep = cache.v[tables[0, page].item(), at].clone()
    cache.v[tables[0, page].item(), at, :, 5] = bad
    got = cache.attend(*args)
    compare(got[:3], want[:3], bound[:3])
    assert not torch.isfinite(got[3:, :, 5].float()).any()
    other = [d for d in range(dim) if d != 5]
    compare(got[..., other], want[..., other], bound[..., other])
    cache.v[tables[0, page].item(), at] = keep
    cache.k[tables[0, page].item(), at, :, 7] = float("nan")
    got = cache.attend(*args)
    compare(got[:3], want[:3], bound[:3])
    assert got[3:].isnan().all()


@pytest.mark.parametrize("nhd", [False, True])
def test_layouts(dev, nhd):
    """Queries that are a view of a wider buffer, an output of wide rows, caches of either order, tables of wide rows; and the same
    bits from copies side by side."""
    gen = torch.Generator().manual_seed(2)
    cache = make_cache(gen, dev, 30, 48, 4, 128, BF, nhd)
    wide = torch.randn((9, 12 * 128 + 64), generator=gen).to(BF).to(dev)
    q = wide[:, :8 * 128].view(9, 8, 128)
    tables = make_tables(gen, dev, [5, 4, 6], 30, 6)
    more = torch.zeros((3, 11), dtype=torch.int32, device=dev)
    more[:, 2:8] = tables
    args = (i32([230, 181, 288], dev), i32([0, 3, 4], dev), i32([3, 1, 5], dev), 5)
    out = torch.full((9, 10 * 128), 5.0, dtype=BF, device=dev)
    cache.attend(q, more[:, 2:8], *args, out=out[:, 128:9 * 128].view(9, 8, 128))
    copy = PagedCache(cache.k.contiguous(), cache.v.contiguous())
    want = copy.attend(q.contiguous(), tables, *args)
    assert torch.equal(out[:, 128:9 * 128].reshape(9, 8, 128).view(torch.int16), want.view(torch.int16))
    assert (out[:, :128] == 5.0).all() and (out[:, 9 * 128:] == 5.0).all()
    odd = torch.zeros((9, 8, 129), dtype=BF, device=dev)[..., 1:]            # rows that start at odd elements: copied
    odd.copy_(q)
    assert torch.equal(copy.attend(odd, tables, *args).view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("n_new", [1, 3, 40])
def test_a_split_makes_rows_their_own(dev, n_new):
    """With pieces of a given size a row's bits are its own, whatever stands beside it, how wide the tables are and how many new
    tokens others have; chosen pieces are the same up to rounding."""
    gen = torch.Generator().manual_seed(n_new)
    lengths = [n_new + v for v in (0, 1000, 255, 2000, 90)]
    cache, q, tables, first, out = batch(gen, dev, lengths, [n_new] * 5, 8, 2, 128, 16, split=256)
    for b in range(5):
        rows = slice(first[b], first[b] + n_new)
        wider = torch.cat([tables[b:b + 1], tables[b:b + 1]], 1).contiguous()
        for t, top in ((tables[b:b + 1], n_new), (wider, n_new + 9)):
            one = cache.attend(q[rows], t, i32(lengths[b:b + 1], dev), i32([0], dev), i32([n_new], dev), top, split=256)
            assert torch.equal(one.view(torch.int16), out[rows].view(torch.int16)), b
    for split in (128, 512, 1 << 20):
        batch(gen, dev, lengths, [n_new] * 5, 8, 2, 128, 16, split=split)


def test_many_requests(dev):
    """More requests than a wave has lanes, padding among them, in tables that could hold far more."""
    gen = torch.Generator().manual_seed(4)
    lengths = [1 + i * 37 % 160 for i in range(150)]
    batch(gen, dev, lengths, [-1 if i % 11 == 3 else 1 for i in range(150)], 4, 2, 64, 16, width=300)
    batch(gen, dev, lengths[:70], [1 + i % 3 for i in range(70)], 4, 2, 64, 16, split=128)


@pytest.mark.parametrize("split", [0, 128])
def test_many_prompts(dev, split):
    """More prompts than a wave has lanes, some of few rows among them, padding, and prompts long enough to be cut."""
    gen = torch.Generator().manual_seed(14)
    n_new = [-1 if i % 13 == 4 else 1 + i * 5 % 19 for i in range(70)]
    batch(gen, dev, [max(n, 0) + i * 11 % 50 for i, n in enumerate(n_new)], n_new, 8, 2, 64, 16, split=split)
    batch(gen, dev, [1500, 40, 900], [20, 20, 1], 8, 2, 128, 32, split=split)


@pytest.mark.parametrize("dim,hq,hkv", [(64, 8, 2), (128, 8, 2), (128, 12, 1), (256, 4, 1)])
@pytest.mark.parametrize("cache_dtype", [BF, E8])
@pytest.mark.parametrize("window", [0, 700])
def test_tokens_beside_prompts(dev, dim, hq, hkv, cache_dtype, window):
    """A batch of prompts, tokens far into their answers (cut into pieces) and drafts; with a split the tokens' bits are those of a
    batch without prompts."""
    gen = torch.Generator().manual_seed(dim + hq + window)
    lengths, n_new = [6000, 430, 3001, 12, 129, 1700], [1, 300, 2, 1, 129, 1]
    batch(gen, dev, lengths, n_new, hq, hkv, dim, 32, BF, cache_dtype, window=window)
    cache, q, tables, first, out = batch(gen, dev, lengths, n_new, hq, hkv, dim, 32, BF, cache_dtype, window=window, split=256)
    few = [0, 2, 3, 5]
    pick = lambda v: i32([v[b] for b in few], dev)  # noqa: E731
    alone = torch.zeros_like(out)
    cache.attend(q, tables[few].contiguous(), pick(lengths), pick(first), pick(n_new), 2, window=window, split=256, out=alone)
    for b in few:
        rows = slice(first[b], first[b] + n_new[b])
        assert torch.equal(alone[rows].view(torch.int16), out[rows].view(torch.int16)), b


def test_one_head_of_the_cache_for_all(dev):
    """A cache that is only read may show one head as many (a stride of zero)."""
    gen = torch.Generator().manual_seed(15)
    one = make_cache(gen, dev, 6, 32, 1, 64, BF)
    wide = PagedCache(*(t.expand(6, 32, 4, 64) for t in (one.k, one.v)))
    q = torch.randn((2, 8, 64), generator=gen).to(BF).to(dev)
    args = (q, i32([[3, 1], [2, 5]], dev), i32([60, 33], dev))
    assert torch.equal(one.attend(*args, split=128), wide.attend(*args, split=128))
    with pytest.raises(RuntimeError, match="overlap"):
        wide.append(q, torch.zeros((2, 4, 64), dtype=BF, device=dev), torch.zeros((2, 4, 64), dtype=BF, device=dev),
                    torch.arange(2, device=dev))


def test_one_long_request(dev):
    gen = torch.Generator().manual_seed(6)
    for lengths, n_new in (([20011], [1]), ([9000, 12], [3, 1])):
        batch(gen, dev, lengths, n_new, 8, 2, 128, 16)
        batch(gen, dev, lengths, n_new, 4, 2, 64, 16, window=5000)


def test_a_cache_past_32_bits(dev):
    """Pages whose elements and bytes lie past 2^31 and 2^32 of their cache."""
    gen = torch.Generator().manual_seed(7)
    pages, page, heads, dim = 150_000, 16, 8, 128             # 2.46e9 elements, 4.9e9 bytes each
    k, v = (torch.empty((pages, heads, page, dim), dtype=BF, device=dev).transpose(1, 2) for _ in range(2))
    cache = PagedCache(k, v)
    T, far = 40, pages - 1
    x = [torch.randn((T, h, dim), generator=gen).to(BF).to(dev) for h in (16, 8, 8)]
    tables = i32([[far, 140_000, far - 1]], dev)
    slots = torch.tensor([int(tables[0, t // page]) * page + t % page for t in range(T)], device=dev)
    q = cache.append(*x, slots)
    assert torch.equal(q, x[0]) and torch.equal(cache.k[far], x[1][:16]) and torch.equal(cache.v[140_000], x[2][16:32])
    small = PagedCache(torch.stack([cache.k[int(p)] for p in tables[0]]), torch.stack([cache.v[int(p)] for p in tables[0]]))
    for n in (1, T):
        args = (i32([T], dev), i32([0], dev), i32([n], dev), n)
        got = cache.attend(q[T - n:], tables, *args)
        assert torch.equal(got, small.attend(q[T - n:], i32([[0, 1, 2]], dev), *args))


def test_graph_and_streams(dev):
    """A captured step (append, then attend) replayed with other tokens, slots, lengths and tables between eager work; the same on two
    streams at once."""
    gen = torch.Generator().manual_seed(8)
    B, hq, hkv, dim, page, width = 5, 8, 2, 128, 16, 40
    rotary = Rotary.of_base(dim, device=dev)
    cache = make_cache(gen, dev, B * width, page, hkv, dim, BF)
    tables = torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width)
    qkv = torch.empty((B, (hq + 2 * hkv) * dim), dtype=BF, device=dev)
    q, k, v = (t.view(B, -1, dim) for t in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
    lengths, slots, positions = i32([0] * B, dev), torch.zeros((B,), dtype=torch.int64, device=dev), torch.zeros((B,), dtype=torch.int64, device=dev)
    turned, out = torch.empty((B, hq, dim), dtype=BF, device=dev), torch.empty((B, hq, dim), dtype=BF, device=dev)

    def fill(step):
        at = torch.tensor([(step * 131 + b * 97) % (width * page) for b in range(B)], device=dev)
        lengths.copy_(at + 1)
        positions.copy_(at)
        slots.copy_(tables.long().gather(1, (at // page)[:, None])[:, 0] * page + at % page)
        qkv.copy_(torch.randn(qkv.shape, generator=gen).to(BF))

    def run(o=out):
        cache.append(q, k, v, slots, positions, rotary, out=turned)
        return cache.attend(turned, tables, lengths, out=o)

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for step in range(1, 6):
        fill(step)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want, bound, _ = paged.attention(turned, paged.cache_values(cache), tables, lengths.tolist(), list(range(B)), [1] * B, dim ** -0.5)
        compare(got, want, bound)
        assert torch.equal(run(torch.empty_like(out)).view(torch.int16), got.view(torch.int16))
    others = [torch.cuda.Stream() for _ in range(2)]
    many = [[] for _ in others]
    for s in others:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, res in zip(others, many):
            with torch.cuda.stream(s):
                res.append(cache.attend(turned, tables, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(r.view(torch.int16), got.view(torch.int16)) for res in many for r in res)


# ---- appends

def check_append(gen, dev, T, hq, hkv, dim, page, dtype=BF, cache_dtype=None, rotary=None, norms=True, nhd=False, axes=1, pads=0,
                 far=5000, in_place=False):
    cache_dtype = cache_dtype or dtype
    pages = -(-2 * T // page) + 1
    cache = make_cache(gen, dev, pages, page, hkv, dim, cache_dtype, nhd)
    before = [cache.k.clone(), cache.v.clone()]
    wide = (torch.randn((T, (hq + 2 * hkv) * dim + 8), generator=gen) * 2).to(dtype).to(dev)
    q, k, v = (t.view(T, -1, dim) for t in wide[:, :-8].split([hq * dim, hkv * dim, hkv * dim], 1))
    x = [t.clone() for t in (q, k, v)]
    slots = torch.randperm(pages * page, generator=gen)[:T]
    if pads:
        slots[torch.randperm(T, generator=gen)[:pads]] = torch.tensor([-1, pages * page, 2 ** 40, -2 ** 40])[torch.arange(pads) % 4]
    slots = slots.to(dev)
    positions = torch.randint(0, far, (T,) if axes == 1 else (axes, T), generator=gen).to(dev)
    weights = [(1 + 0.2 * torch.randn((dim,), generator=gen)).to(dtype).to(dev) if norms else None for _ in range(2)]
    out = cache.append(q, k, v, slots, positions, rotary, *weights, out=q if in_place else None)
    assert (out is q) == in_place
    assert torch.equal(wide[:, hq * dim:], torch.cat([x[1].flatten(1), x[2].flatten(1), wide[:, -8:]], 1))
    if not in_place:
        assert torch.equal(q, x[0])
    want = paged.turned(x[0], weights[0], positions, rotary, 1e-6)
    compare(out, want, paged.turned_bound(x[0], weights[0], want, dtype))
    kept = ((slots >= 0) & (slots < pages * page)).cpu()
    s = slots.cpu()[kept]
    for i, (c, old) in enumerate(((cache.k, before[0]), (cache.v, before[1]))):
        want = paged.turned(x[1], weights[1], positions, rotary, 1e-6) if i == 0 else x[2].double().cpu()
        want = want[kept]
        slack = paged.turned_bound(x[1][kept.to(dev)], weights[1], want, torch.float32) if i == 0 else torch.zeros_like(want)
        if cache_dtype == E8:
            scale = cache.k_scale if i == 0 else cache.v_scale
            top = 448.0 * scale.double().cpu()[:, None]
            want = want.clamp(-top, top)
            bound = paged.e4m3_bound(want, scale, slack)
        else:
            bound = paged.turned_bound(None, None, want, dtype) if i == 0 else torch.full_like(want, 1e-300)
        compare(paged.cache_values(cache)[i][s // page, s % page], want, bound)
        bits = torch.uint8 if cache_dtype == E8 else torch.int16
        same = torch.ones((pages, page), dtype=torch.bool)
        same[s // page, s % page] = False
        assert torch.equal(c.view(bits)[same.to(dev)], old.view(bits)[same.to(dev)])
    return out


@pytest.mark.parametrize("T", [1, 3, 33, 1023, 1024, 1027])
@pytest.mark.parametrize("dim,hq,hkv", [(128, 32, 4), (64, 3, 1), (256, 16, 2), (64, 12, 4)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_append(dev, T, dim, hq, hkv, dtype):
    gen = torch.Generator().manual_seed(T)
    check_append(gen, dev, T, hq, hkv, dim, 16, dtype, rotary=Rotary.of_base(dim, device=dev))


@pytest.mark.parametrize("T", [5, 1100])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("part", [1, 2, 4])
def test_append_rotations(dev, T, dim, adjacent, part):
    """Either pairing, any share of a head, with and without norms, several axes, padding, in place and not."""
    gen = torch.Generator().manual_seed(part)
    n = dim // part
    for i, axes in enumerate((1, 3)):
        half = n // 2
        sections = None if axes == 1 else [half - 2 * (half // 4), half // 4, half // 4]
        rotary = Rotary.of_base(n, 500000.0, sections, interleaved=adjacent, device=dev, adjacent=adjacent, scale=1.25)
        check_append(gen, dev, T, 5, 2, dim, 48, rotary=rotary, norms=i == 0, axes=axes, pads=4, in_place=i == 1, nhd=adjacent)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("T", [7, 1100])
def test_append_eight_bits(dev, dtype, dim, T):
    gen = torch.Generator().manual_seed(T)
    check_append(gen, dev, T, 4, 4, dim, 80, dtype, E8, Rotary.of_base(dim, device=dev), pads=2)


def test_append_without_a_rotation(dev):
    gen = torch.Generator().manual_seed(1)
    for norms in (False, True):
        check_append(gen, dev, 20, 4, 2, 128, 16, norms=norms)


def test_append_far_positions(dev):
    """Angles past what 32 bits keep the fraction of."""
    gen = torch.Generator().manual_seed(2)
    check_append(gen, dev, 64, 2, 1, 128, 16, rotary=Rotary.of_base(128, device=dev), far=2 ** 31)


def test_append_eight_bits_at_their_ends(dev):
    """Beyond the largest value, infinities, NaN, ties and subnormal values."""
    dim, s = 64, 0.5
    cache = PagedCache.empty(1, 16, 1, dim, E8, dev, k_scale=s, v_scale=s)
    vals = [448, 449, 464, 1e4, float("inf"), -448, -500, -float("inf"), float("nan"), 1.0625, 1.1875, -1.0625, 2 ** -9, 2 ** -10,
            3 * 2 ** -10, 2 ** -11, 0.0, -0.0, 2 ** -6, 0.9375 * 2 ** -6, 17, 19]
    want = [448, 448, 448, 448, 448, -448, -448, -448, float("nan"), 1.0, 1.25, -1.0, 2 ** -9, 0.0, 2 ** -8, 0.0, 0.0, 0.0, 2 ** -6,
            0.9375 * 2 ** -6 + 2 ** -10, 16, 20]
    want[19] = float((torch.tensor([0.9375 * 2 ** -6]).to(E8)).float())
    x = torch.zeros((1, 1, dim), dtype=HF)
    x[0, 0, :len(vals)] = torch.tensor(vals) * s
    cache.append(x.to(dev), x.to(dev), x.to(dev), torch.tensor([3], device=dev))
    for c in (cache.k, cache.v):
        got = c[0, 3, 0, :len(vals)].float().cpu()
        assert torch.equal(got.nan_to_num(nan=-1.0), torch.tensor(want).float().nan_to_num(nan=-1.0)), got


def test_append_rows_are_their_own(dev):
    """A row's bits in a prompt are those of the row alone."""
    gen = torch.Generator().manual_seed(9)
    T, dim, page = 1500, 128, 16
    rotary = Rotary.of_base(dim, device=dev)
    x = [torch.randn((T, h, dim), generator=gen).to(BF).to(dev) for h in (8, 2, 2)]
    w = [torch.randn((dim,), generator=gen).to(BF).to(dev) for _ in range(2)]
    slots, positions = torch.arange(T, device=dev), torch.arange(T, device=dev) * 3
    a, b = (PagedCache.empty(100, page, 2, dim, device=dev) for _ in range(2))
    whole = a.append(*x, slots, positions, rotary, *w)
    for lo, hi in ((0, 1), (1, 4), (4, 900), (900, 1500)):
        part = b.append(*(t[lo:hi] for t in x), slots[lo:hi], positions[lo:hi], rotary, *w)
        assert torch.equal(part.view(torch.int16), whole[lo:hi].view(torch.int16))
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_none_at_all(dev):
    """No rows and no requests are no error."""
    cache = PagedCache.empty(2, 16, 1, 64, device=dev)
    none = torch.zeros((0, 2, 64), dtype=BF, device=dev)
    assert cache.append(none, none[:, :1], none[:, :1], torch.zeros((0,), dtype=torch.int64, device=dev)).shape == none.shape
    assert cache.attend(none, i32([[0]], dev), i32([3], dev), i32([0], dev), i32([0], dev)).shape == none.shape
    q = torch.ones((2, 2, 64), dtype=BF, device=dev)
    out = torch.full_like(q, 2.0)
    cache.attend(q, torch.zeros((0, 4), dtype=torch.int32, device=dev), i32([], dev), out=out)
    assert (out == 2.0).all()


def test_refusals(dev):
    """What the extension refuses before it launches anything."""
    cache = PagedCache.empty(4, 16, 2, 64, device=dev)
    q, kv, slots = torch.zeros((3, 4, 64), dtype=BF, device=dev), torch.zeros((3, 2, 64), dtype=BF, device=dev), torch.arange(3, device=dev)
    tables, lengths = i32([[0], [1], [2]], dev), i32([1, 2, 3], dev)
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q.half()), dict(k=kv[:2]), dict(k=kv[:, :1]), dict(slots=slots.int()),
                dict(slots=slots[:2]), dict(slots=slots.cpu()), dict(positions=slots, rotary=Rotary.of_base(128, device=dev)),
                dict(rotary=Rotary.of_base(64, device=dev)), dict(positions=slots[:2], rotary=Rotary.of_base(64, device=dev)),
                dict(positions=torch.stack([slots] * 2), rotary=Rotary.of_base(64, device=dev)),
                dict(q_norm=torch.ones((32,), dtype=BF, device=dev)), dict(k_norm=torch.ones((64,), device=dev)), dict(out=q[:2]),
                dict(q=q[..., :64], out=torch.zeros((3, 8, 64), dtype=BF, device=dev)[:, ::3])):
        args = {**dict(q=q, k=kv, v=kv, slots=slots), **bad}
        with pytest.raises(RuntimeError):
            cache.append(**args)
    buf = torch.zeros((3, 8, 64), dtype=BF, device=dev)
    with pytest.raises(RuntimeError, match="overlaps"):
        cache.append(buf[:, :4], buf[:, 4:6], buf[:, 6:], slots, out=buf[:, 2:6])
    with pytest.raises(RuntimeError, match="overlaps"):
        cache.append(q, buf[:, 4:6], buf[:, 6:], slots, out=buf[:, 3:7])
    for bad in (dict(q=q.half()), dict(q=torch.zeros((3, 3, 64), dtype=BF, device=dev)), dict(tables=tables.long()),
                dict(tables=tables[:, :0]), dict(tables=tables.cpu()), dict(lengths=lengths[:2]), dict(lengths=lengths.long()),
                dict(first=lengths[:2]), dict(n_new=lengths.long()), dict(max_new=2), dict(max_new=0), dict(scale=0.0), dict(scale=-1.0), dict(window=-1),
                dict(split=100), dict(split=-128), dict(out=q), dict(out=q.half())):
        args = {**dict(q=q, tables=tables, lengths=lengths), **bad}
        with pytest.raises(RuntimeError):
            cache.attend(**args)
