"""GPU checks of the attention over a paged cache where one key has nearly all of a row's weight and a value of next to nothing, and the
row's output is the sum of thousands of weights some 2^-20 to 2^-27 of the largest: fp16's own rounding of such weights must not show.

Bars are paged.attention's: every weight is off by at most half a step of itself, which fp16 weights are down to 2^-27 of the largest; below
that they are off by at most 2^-38 of it, which is added here."""
import pytest
import torch

import paged
from test_gpu_attention import compare, i32
from vllm_espalier.attention import PagedCache

pytestmark = pytest.mark.gpu
BF, HF, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def one_heavy_key(dev, dim, dtype, cache_dtype, keys, n_new, below, heavy=3, hq=2):
    """(cache, q, table): `keys` keys of one head whose weights are about 2^-below of key `heavy`'s for every row; their values are about
    100 and its own is 0."""
    gen = torch.Generator().manual_seed(keys + int(below))
    page = 64
    pages = -(-keys // page) + 1
    q = torch.randn((n_new, hq, dim), generator=gen) * 0.02
    q[..., 0] = 8.0
    half = below / 1.4426950408889634 / 8.0 * dim ** 0.5 / 2
    k, v = torch.randn((2, pages, 1, page, dim), generator=gen) * 0.05
    v = 100.0 + 20.0 * v
    order = torch.randperm(pages - 1, generator=gen) + 1
    k[..., 0] = -half
    k[order[heavy // page], 0, heavy % page, 0] = half
    v[order[heavy // page], 0, heavy % page] = 0.0
    scale = None
    if cache_dtype == E8:                                     # (its keys' first elements are the largest value of eight bits)
        scale = [torch.tensor([s], dtype=torch.float32, device=dev) for s in (half / 448.0, 0.5)]
        k, v = k / scale[0].cpu(), v / 0.5
    cache = PagedCache(*(t.to(cache_dtype).to(dev).transpose(1, 2) for t in (k, v)), *(scale or ()))
    return cache, q.to(dtype).to(dev), order[None].to(torch.int32).to(dev)


@pytest.mark.parametrize("below", [20.4, 21.6, 24.6, 26.0, 31.0])
@pytest.mark.parametrize("dtype,cache_dtype", [(HF, HF), (HF, E8), (BF, BF)])
@pytest.mark.parametrize("dim,n_new,keys,splits", [(64, 1, 20000, (0, 128, 1 << 20)), (128, 1, 20000, (0, 1 << 20)), (256, 2, 9000, (0, 1 << 20)),
                                                   (64, 70, 6000, (0, 128)), (128, 70, 6000, (0, 128)), (256, 70, 6000, (0, 128))])
def test_small_weights(dev, dim, n_new, keys, splits, dtype, cache_dtype, below):
    cache, q, table = one_heavy_key(dev, dim, dtype, cache_dtype, keys, n_new, below)
    kv = paged.cache_values(cache)
    want, bound, _ = paged.attention(q, kv, table, [keys], [0], [n_new], dim ** -0.5)
    assert float(want.abs().min()) > 0.25 * (keys - n_new) * 100.0 * 2.0 ** -below      # (the sums are what they were made to be)
    if dtype == HF:
        bound = bound + 2.0 ** -38 * keys * float(kv[1].abs().max())
    for split in splits:
        got = cache.attend(q, table, i32([keys], dev), i32([0], dev), i32([n_new], dev), n_new, split=split)
        compare(got, want, bound)


@pytest.mark.parametrize("n_new", [1, 70])
def test_scores_that_grow(dev, n_new):
    """Every key heavier than those before it, by little and by much: the weights' base moves all the time, and no weight leaves fp16."""
    gen = torch.Generator().manual_seed(n_new)
    dim, keys, page = 128, 3000, 16
    pages = -(-keys // page)
    q = torch.randn((n_new, 2, dim), generator=gen) * 0.3
    q[..., 0] = 4.0
    for step in (0.003, 0.02, 0.3):
        k, v = torch.randn((2, pages, 1, page, dim), generator=gen)
        k[:, 0, :, 0] = (step * torch.arange(pages * page) * dim ** 0.5 / 4.0).view(pages, page) - 100.0
        cache = PagedCache(*(t.to(HF).to(dev).transpose(1, 2) for t in (k, v * 500.0)))
        x, table = q.to(HF).to(dev), torch.arange(pages, dtype=torch.int32, device=dev)[None]
        kv = paged.cache_values(cache)
        want, bound, _ = paged.attention(x, kv, table, [keys], [0], [n_new], dim ** -0.5)
        bound = bound + 2.0 ** -38 * keys * float(kv[1].abs().max())
        for split in (0, 1 << 20):
            compare(cache.attend(x, table, i32([keys], dev), i32([0], dev), i32([n_new], dev), n_new, split=split), want, bound)


@pytest.mark.parametrize("n_new", [1, 70])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [100.0, 300.0, 1000.0, 3000.0])
def test_large_scores(dev, n_new, sign, size):
    """Scores of up to 2^26 over the weights' exponents, of either sign: the keys that are far above the others share all of the weight,
    whatever they come behind (all others' exponents are smaller by thousands)."""
    gen = torch.Generator().manual_seed(int(size))
    dim, keys, page = 64, 1200, 16
    pages = -(-keys // page)
    q = torch.full((n_new, 2, dim), size)
    k = torch.full((pages, 1, page, dim), size * 0.5 * sign)
    flat = k.view(-1, dim)
    flat[40:] += size * 0.125 * sign                          # rising, or falling, in two steps
    flat[[700, 900]] += size * 0.125 * sign
    v = torch.randn((pages, 1, page, dim), generator=gen) * 50.0
    cache = PagedCache(*(t.to(HF).to(dev).transpose(1, 2) for t in (k, v)))
    x, table = q.to(HF).to(dev), torch.arange(pages, dtype=torch.int32, device=dev)[None]
    values = v.to(HF).double().view(-1, dim)
    want = (values[[700, 900]] if sign > 0 else values[:40]).mean(0).expand(n_new, 2, dim)
    # equal weights, off by half a step each, as the output is; the sums' 2^-18
    bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -18) * values.abs().max() + torch.finfo(HF).tiny
    for split in (0, 128, 1 << 20):
        got = cache.attend(x, table, i32([keys], dev), i32([0], dev), i32([n_new], dev), n_new, split=split)
        compare(got, want, bound)
