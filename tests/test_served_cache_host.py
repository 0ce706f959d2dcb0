"""Checks on the CPU of what a served cache is made of: caches whose keys and values share memory, rotations whose axes' shares do not fit,
and the synthetic decoder's bookkeeping around its caches."""
import ctypes
import itertools
import random
import re
from pathlib import Path

import pytest
import torch

from test_attention_host import Cache, FAR, lib  # noqa: F401
from vllm_espalier import step as S
from vllm_espalier.attention import Rotary


def append(lib, k, v, strides, pages, page, heads, dim, dtype=1):  # noqa: F811
    """No rows into this cache: 0, or 1 where it is refused. strides: of pages, tokens and heads, k's and v's alike."""
    scales = (16, 16) if dtype == 3 else (None, None)
    cache = Cache(k, v, dtype, pages, page, heads, dim, *strides, *strides, *scales)
    return lib.esp_cache_append(None, 0, 0, None, 0, 0, None, 0, 0, 0, heads, 1, ctypes.byref(cache), None, None, 0, 1, None, None, 0, 0, 1.0,
                                None, None, 1e-6, None, 0, 0, None)


def test_keys_and_values_apart(lib):  # noqa: F811
    """Two tensors, two halves of one (by pages, tokens, heads or whole), and what shares an element."""
    page, heads, dim = 16, 2, 64
    for dtype, size in ((1, 2), (3, 1)):
        for k, v in itertools.permutations((FAR, 9 * FAR)):
            assert append(lib, k, v, (2048, 64, 1024), 8, page, heads, dim, dtype) == 0
        plain = 8 * 2048                                       # elements of one alone
        for between, strides, what in (
                (plain, (2048, 64, 1024), "one after the other"), (2048, (4096, 64, 1024), "a page of each in turn"),
                (128, (4096, 256, 64), "a token of each in turn"), (64, (4096, 256, 128), "a head of each in turn"),
                (1024, (4096, 64, 2048), "a page's head of each in turn")):
            for sign in (1, -1):
                assert append(lib, FAR, FAR + sign * between * size, strides, 8, page, heads, dim, dtype) == 0, what
        for between, strides in ((0, (2048, 64, 1024)), (2048, (2048, 64, 1024)), (7 * 2048, (2048, 64, 1024)), (64, (2048, 64, 1024)),
                                 (3 * 2048 + 1024 + 5 * 64, (2048, 64, 1024)), (4096, (4096, 64, 1024)), (256, (4096, 256, 64)),
                                 (7 * 2048 + 1024 + 960 + 32, (2048, 64, 1024))):
            for sign in (1, -1):
                assert append(lib, FAR, FAR + sign * between * size, strides, 8, page, heads, dim, dtype) == 1, (between, strides)
                assert "k and v" in lib.esp_last_error().decode()


def test_keys_and_values_apart_by_enumeration(lib):  # noqa: F811
    """The same of small caches of many layouts against all of their places."""
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(600):
        page, dim = 16, 64
        pages, heads = rng.choice([1, 2, 3]), rng.choice([1, 2, 3])
        order, strides, span = rng.sample([("page", pages), ("token", page), ("head", heads)], 3), {}, dim
        for name, n in order:
            strides[name] = span + rng.choice([0, 0, 64, 128, span])
            span = strides[name] * (n - 1) + span if n > 1 else span
        if strides["token"] < dim:
            continue
        at = {p * strides["page"] + t * strides["token"] + h * strides["head"] for p in range(pages) for t in range(page) for h in range(heads)}
        for _ in range(4):
            between = rng.choice([rng.randrange(-span // 8, span // 8) * 8, rng.choice(list(at)) - rng.choice(list(at)), strides[order[-1][0]] // 128 * 64])
            starts = {a // 8 + i for a in at for i in range(dim // 8)}
            want = any(a + between // 8 in starts for a in starts)
            got = append(lib, 1 << 30, (1 << 30) + between * 2, (strides["page"], strides["token"], strides["head"]), pages, page, heads, dim)
            assert got == int(want), (order, strides, between)
            seen[got] += 1
    assert min(seen) > 100, seen


def test_interleaved_shares():
    """Every axis has as many pairs as it was given, or the rotation is refused."""
    for sections in ([16, 8, 8], [12, 10, 10], [32], [16, 16], [11, 11, 10], [32, 0, 0], [20, 2, 10], [8, 8, 8, 8], [17, 5, 5, 5]):
        axes = Rotary.of_base(64, sections=sections, interleaved=True, device="cpu").axes
        assert [int((axes == a).sum()) for a in range(len(sections))] == sections
        assert all(a in (0, f % len(sections)) for f, a in enumerate(axes.tolist()))
    for sections in ([4, 14, 14], [0, 16, 16], [10, 11, 11], [15, 17], [7, 9, 8, 8], [0, 32]):
        with pytest.raises(ValueError, match="turns"):
            Rotary.of_base(64, sections=sections, interleaved=True, device="cpu")
        axes = Rotary.of_base(64, sections=sections, device="cpu").axes                  # (one axis after the other any shares fit)
        assert [int((axes == a).sum()) for a in range(len(sections))] == sections


@pytest.fixture(scope="module")
def decoder():
    return S.SyntheticDecoder(n_layers=2, seed=9, device="cpu", E=4, vocab=1024)


def test_no_places_without_caches(decoder):
    with pytest.raises(RuntimeError, match="use_cache"):
        decoder.sequences(decoder.buffers(3))


def test_places_belong_to_the_caches(decoder):
    """None of the former caches' pages after others have come."""
    b = decoder.buffers(3)
    decoder.use_cache(4, 32)
    s = decoder.sequences(b, max_new=3)
    s.place([[1, 2]], [34], [3])
    assert s.page == 32 and s.slots.tolist() == [63, 64, 65]
    assert b.sequences is s
    decoder.use_cache(8, 16)
    with pytest.raises(RuntimeError, match="sequences"):
        decoder._mixed(decoder.layers[0], b)
    assert decoder.sequences(b).page == 16 and b.sequences.tables.shape == (3, 8)


def test_algorithmic_bytes_count_the_norms_of_q_and_k():
    dec = S.SyntheticDecoder(n_layers=2, seed=9, device="cpu", E=4, vocab=1024)
    picks = [torch.empty((0,), dtype=torch.int32)] * 2
    plain = dec.algorithmic_bytes(picks, 3)
    dec.use_cache(4, 32)
    assert dec.algorithmic_bytes(picks, 3) - plain == 2 * 2 * S.HEAD_DIM * 2
    dec.layers[1].cache = None                                # a layer without a cache reads none of them
    assert dec.algorithmic_bytes(picks, 3) - plain == 2 * S.HEAD_DIM * 2


def test_the_largest_vocabulary_is_the_headers(lib):  # noqa: F811
    """What include/espalier.h says of V, the scratch's size and the call's own check are one number."""
    text = (Path(__file__).resolve().parent.parent / "include" / "espalier.h").read_text()
    most = 1 << int(re.search(r"R < 2\^31, V <= 2\^(\d+), R \* ceil", text).group(1))
    call = lambda V: lib.esp_token_logprobs(FAR, 1, V, 1, V, 16, None, 0, 16, None, None, None, None, 16, 0, None)  # noqa: E731
    assert lib.esp_token_logprobs_scratch(1, most, 0) > 0 and lib.esp_token_logprobs_scratch(1, most + 1, 0) == 0
    assert call(most) == 1 and "scratch" in lib.esp_last_error().decode()
    assert call(most + 1) == 1 and "V" in lib.esp_last_error().decode()
