"""Refusals of the paged cache's appends, the attention over it and the token log-probabilities, on the CPU: the C ABI's argument
checks fail with a code and a message before any HIP call; what Rotary and PagedCache check; what the plain forms of the tests say."""
import ctypes
from pathlib import Path

import pytest
import torch

import paged
from vllm_espalier import step as S
from vllm_espalier.attention import PagedCache, Rotary

LIB = Path(__file__).resolve().parent.parent / "vllm-espalier_amd" / "vllm_espalier" / "libespalier_hip.so"
P, I64, INT, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double
FAR = 1 << 24                                                 # made-up addresses, far apart


class Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("dtype", INT), ("pages", I64), ("page", I64), ("heads", I64), ("dim", I64), ("k_page", I64),
                ("k_token", I64), ("k_head", I64), ("v_page", I64), ("v_token", I64), ("v_head", I64), ("k_scale", P), ("v_scale", P)]


@pytest.fixture(scope="module")
def lib(ext):
    L = ctypes.CDLL(str(LIB))
    C = ctypes.POINTER(Cache)
    L.esp_last_error.restype = ctypes.c_char_p
    L.esp_cache_append.argtypes = [P, I64, I64] * 3 + [I64, I64, INT, C, P, P, I64, I64, P, P, I64, INT, F64, P, P, F64, P, I64, I64, P]
    L.esp_paged_attention.argtypes = [P, I64, I64, I64, I64, INT, C, P, I64, I64, P, P, P, I64, I64, F64, I64, I64, P, I64, I64, P, I64, P]
    L.esp_paged_attention_scratch.argtypes, L.esp_paged_attention_scratch.restype = [I64, I64, I64, I64, C, I64, I64], I64
    L.esp_token_logprobs.argtypes = [P, INT, I64, I64, I64, P, P, I64, P, P, P, P, P, P, I64, P]
    L.esp_token_logprobs_scratch.argtypes, L.esp_token_logprobs_scratch.restype = [I64] * 3, I64
    return L


def _cache(over):
    c = dict(k=8 * FAR, v=9 * FAR, dtype=1, pages=8, page=16, heads=2, dim=64, k_page=2048, k_token=64, k_head=1024, v_page=2048,
             v_token=64, v_head=1024, k_scale=None, v_scale=None)
    c.update({n: over.pop(n) for n in list(over) if n in c})
    return Cache(**c)


CACHE_ERRORS = [
    (dict(dtype=0), "dtype or e4m3"), (dict(dtype=2), "dtype or e4m3"), (dict(dim=96), "64, 128 or 256"), (dict(dim=0), "64, 128 or 256"),
    (dict(heads=0), "heads"), (dict(heads=2000), "heads"), (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"), (dict(page=8), "pages"),
    (dict(page=24), "pages"), (dict(page=0), "pages"), (dict(page=1 << 20), "pages"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(dtype=3), "scale"), (dict(k_scale=16, v_scale=16), "scale"), (dict(dtype=3, k_scale=16), "scale"), (dict(k=8 * FAR + 8), "aligned"),
    (dict(k_token=68), "aligned"), (dict(v_head=1028), "aligned"), (dict(v_page=-2048), "strides"), (dict(k_token=56), "overlap"),
    (dict(v_token=32), "overlap"), (dict(k_token=1 << 24), "at most 2^24"), (dict(dtype=3, k_scale=16, v_scale=16, k_token=72), "aligned")]


def test_overlapping_caches(lib):
    """A cache that is written must lie apart: pages, tokens and heads in any order, but none over another."""
    for over in (dict(k_head=0), dict(v_head=48), dict(k_page=1024), dict(v_page=0), dict(k_token=128, k_head=64, k_page=1024),
                 dict(v_token=64, v_head=1024, v_page=2040)):
        assert _append(lib, **over) == 1 and "overlap" in lib.esp_last_error().decode(), over
    for over in (dict(k_token=128, k_head=64), dict(k_page=64, k_token=512, k_head=8192), dict(heads=1, k_head=0, v_head=0, kr=64, vr=64),
                 dict(pages=1, k_page=0, v_page=0)):
        assert _append(lib, T=0, **over) == 0, (over, lib.esp_last_error())
    assert _attend(lib, T=0, k_head=0, v_head=0) == 0          # what is only read may be one head for all


def _append(lib, **over):
    cache = _cache(over)
    a = dict(q=FAR, qr=256, qh=64, k_rows=2 * FAR, kr=128, kh=64, v_rows=3 * FAR, vr=128, vh=64, T=4, Hq=4, rows=1, slots=16, pos=16, axis=4,
             n_axes=1, freq=16, axes=None, half=32, wq=16, wk=16, out=4 * FAR, outr=256, outh=64)
    a.update(over)
    return lib.esp_cache_append(a["q"], a["qr"], a["qh"], a["k_rows"], a["kr"], a["kh"], a["v_rows"], a["vr"], a["vh"], a["T"], a["Hq"],
                                a["rows"], ctypes.byref(cache), a["slots"], a["pos"], a["axis"], a["n_axes"], a["freq"], a["axes"],
                                a["half"], 0, 1.0, a["wq"], a["wk"], 1e-6, a["out"], a["outr"], a["outh"], None)


@pytest.mark.parametrize("over,needle", CACHE_ERRORS + [
    (dict(rows=2), "bf16 or fp16"), (dict(T=-1), "rows"), (dict(T=1 << 24), "rows"), (dict(Hq=-1), "heads"), (dict(Hq=1025), "heads"),
    (dict(half=12), "multiple of 8"), (dict(half=40), "half a head"), (dict(half=-8), "multiple of 8"), (dict(n_axes=0), "axes"),
    (dict(n_axes=17), "axes"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(k_rows=None), "null"), (dict(slots=None), "null"),
    (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(n_axes=3), "axis of each"), (dict(n_axes=3, axes=16, axis=3), "overlap"),
    (dict(qr=260), "multiples of 8"), (dict(vh=-64), "multiples of 8"), (dict(kr=1 << 32), "below"), (dict(q=FAR + 8), "aligned"),
    (dict(wk=24), "aligned"), (dict(outh=56), "overlap"), (dict(outr=248), "overlap"), (dict(out=FAR + 128), "overlaps q"),
    (dict(out=FAR, outr=512), "overlaps q"), (dict(out=2 * FAR), "overlaps k or v"), (dict(out=3 * FAR + 768), "overlaps k or v")])
def test_append_argument_errors(lib, over, needle):
    assert _append(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def _attend(lib, **over):
    cache = _cache(over)
    a = dict(q=FAR, qr=256, qh=64, T=4, Hq=4, rows=1, tables=16, tr=8, width=8, lengths=16, first=16, n=16, B=2, new=2, scale=0.1, window=0,
             split=0, out=4 * FAR, outr=256, outh=64, scratch=16, bytes=1 << 40)
    a.update(over)
    return lib.esp_paged_attention(a["q"], a["qr"], a["qh"], a["T"], a["Hq"], a["rows"], ctypes.byref(cache), a["tables"], a["tr"],
                                   a["width"], a["lengths"], a["first"], a["n"], a["B"], a["new"], a["scale"], a["window"], a["split"],
                                   a["out"], a["outr"], a["outh"], a["scratch"], a["bytes"], None)


@pytest.mark.parametrize("over,needle", CACHE_ERRORS + [
    (dict(rows=2), "bf16 or fp16"), (dict(T=-1), "rows"), (dict(T=1 << 24), "rows"), (dict(B=-1), "requests"), (dict(B=(1 << 20) + 1), "requests"),
    (dict(Hq=3), "multiple"), (dict(Hq=0), "multiple"), (dict(Hq=1 << 17), "multiple"), (dict(new=0), "new tokens"), (dict(new=1 << 24), "new tokens"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(window=-1), "window"), (dict(window=1 << 30), "window"), (dict(split=64), "split"), (dict(split=-128), "split"), (dict(split=1 << 30), "split"),
    (dict(width=-1), "tables"), (dict(width=(1 << 24) + 1, tr=1 << 25), "tables"), (dict(width=0), "at least one page"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(tables=None), "null"), (dict(lengths=None), "null"), (dict(scratch=None), "null"),
    (dict(first=None), "first rows"), (dict(Hq=1 << 16, T=(1 << 24) - 1, heads=1 << 10, qr=0, outr=1 << 31), "rows of heads"), (dict(tr=7), "overlap"), (dict(qr=260), "multiples of 8"), (dict(outh=-64), "multiples of 8"), (dict(out=4 * FAR + 8), "aligned"),
    (dict(scratch=24), "aligned"), (dict(outh=32), "overlap"), (dict(outr=192), "overlap"), (dict(out=FAR), "overlaps q"),
    (dict(out=FAR + 1024), "overlaps q"), (dict(new=(1 << 23) + 1), "rows a request"), (dict(bytes=15), "scratch"),
    (dict(width=1 << 24, tr=1 << 24, split=128, B=1 << 10), "pieces")])
def test_attend_argument_errors(lib, over, needle):
    assert _attend(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def test_rows_of_a_request_stay_countable(lib):
    """Rows a request and head of the cache are told apart by reciprocals in fp32: 2^23 are refused, one fewer not for that."""
    heads = dict(Hq=4, heads=1, outr=256, bytes=15)
    assert _attend(lib, new=1 << 21, **heads) == 1 and "rows a request" in lib.esp_last_error().decode()
    assert _attend(lib, new=(1 << 21) - 1, **heads) == 1 and "scratch" in lib.esp_last_error().decode()


def test_no_rows_is_no_call(lib):
    assert _append(lib, T=0, q=None, k_rows=None, v_rows=None, out=None) == 0
    assert _attend(lib, T=0, q=None, out=None) == 0
    assert _attend(lib, B=0, tables=None, lengths=None) == 0
    assert _logprobs(lib, R=0, logits=None) == 0


def test_attend_scratch(lib):
    """Scratch for every piece of a tile that can have several: at most as many as the lengths' choice makes, none without any."""
    c = Cache(dim=128, heads=4, page=16)
    size = lambda B, new, Hq, width, split: lib.esp_paged_attention_scratch(B, B * new, new, Hq, ctypes.byref(c), width, split)  # noqa: E731
    assert size(1, 1, 32, 8, 0) == 16                          # 128 keys: one piece
    assert size(4, 1, 32, 64, 128) >= 4 * 4 * 8 * 16 * 130 * 4
    assert size(1, 1, 32, 1 << 13, 0) >= 512 * 16 * 130 * 4
    assert size(64, 1, 32, 1 << 13, 0) >= 1024 * 16 * 130 * 4
    assert size(2, 100, 32, 1 << 10, 0) >= 1024 * (32 + 128) * 130 * 4
    assert size(2, 100, 32, 1 << 10, 256) == 16 + 2 * 4 * 64 * 32 * 130 * 4           # prompts are not cut then
    for bad in ((0, 1, 32, 8, 0), (1, 0, 32, 8, 0), (1, 1, 30, 8, 0), (1, 1, 32, -1, 0), (1, 1, 32, 8, 100), (1, 1, 32, 1 << 25, 0)):
        assert size(*bad) == 0


def _logprobs(lib, **over):
    a = dict(logits=FAR, dtype=1, stride=64, R=8, V=64, tokens=16, temp=None, top=5, lp=16, ranks=16, ent=16, ids=16, tlp=16, scratch=16,
             bytes=1 << 40)
    a.update(over)
    return lib.esp_token_logprobs(a["logits"], a["dtype"], a["stride"], a["R"], a["V"], a["tokens"], a["temp"], a["top"], a["lp"],
                                  a["ranks"], a["ent"], a["ids"], a["tlp"], a["scratch"], a["bytes"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(dtype=3), "dtype"), (dict(R=-1), "rows"), (dict(R=1 << 31), "rows"), (dict(V=0), "V"), (dict(V=(1 << 20) + 1), "V"), (dict(top=65), "alternatives"),
    (dict(top=-1), "alternatives"), (dict(V=4, top=5), "alternatives"), (dict(R=1 << 24), "blocks"), (dict(logits=None), "null"),
    (dict(tokens=None), "null"), (dict(lp=None), "null"), (dict(ids=None), "null"), (dict(tlp=None), "null"), (dict(scratch=None), "null"),
    (dict(stride=63), "overlap"), (dict(logits=FAR + 1), "aligned"), (dict(logits=FAR + 2, dtype=2), "aligned"), (dict(scratch=24), "aligned"),
    (dict(bytes=100), "scratch")])
def test_logprobs_argument_errors(lib, over, needle):
    assert _logprobs(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def test_logprobs_scratch(lib):
    assert lib.esp_token_logprobs_scratch(4, 151936, 20) >= 4 * 149 * 16
    assert lib.esp_token_logprobs_scratch(0, 100, 0) == 0 and lib.esp_token_logprobs_scratch(4, 0, 0) == 0


def test_rotary():
    r = Rotary.of_base(64, 1e6, sections=[16, 8, 8], device="cpu")
    assert r.inv_freq.dtype == torch.float64 and torch.allclose(r.inv_freq, 1e6 ** (-torch.arange(32).double() / 32))
    assert r.axes.tolist() == [0] * 16 + [1] * 8 + [2] * 8 and not r.adjacent
    turns = Rotary.of_base(64, sections=[16, 8, 8], interleaved=True, device="cpu", adjacent=True, scale=2.0)
    assert turns.axes.tolist() == [0, 1, 2] * 8 + [0] * 8 and turns.adjacent and turns.scale == 2.0
    assert Rotary.of_base(32, device="cpu").axes is None
    for bad in (lambda: Rotary.of_base(24, device="cpu"), lambda: Rotary.of_base(0, device="cpu"),
                lambda: Rotary.of_base(64, sections=[16, 8], device="cpu"), lambda: Rotary.of_base(64, sections=[40, -8], device="cpu"),
                lambda: Rotary(torch.ones((8,))), lambda: Rotary(torch.ones((12,), dtype=torch.float64)),
                lambda: Rotary(torch.ones((8,), dtype=torch.float64), axes=torch.zeros((8,))),
                lambda: Rotary(torch.ones((8,), dtype=torch.float64), axes=torch.zeros((4,), dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()


def test_paged_cache():
    c = PagedCache.empty(3, 32, 2, 64, device="cpu")
    assert c.k.shape == (3, 32, 2, 64) and c.k.stride() == (4096, 64, 2048, 1) and c.k_scale is None
    e = PagedCache.empty(3, 16, 2, 128, torch.float8_e4m3fn, "cpu", k_scale=0.5, v_scale=[0.25, 2.0])
    assert e.k_scale.tolist() == [0.5, 0.5] and e.v_scale.tolist() == [0.25, 2.0]
    k = torch.zeros((3, 16, 2, 64))
    one = torch.ones((2,))
    for bad in (lambda: PagedCache(k, k), lambda: PagedCache(k.half(), k.bfloat16()), lambda: PagedCache(k.half(), k[:2].half()),
                lambda: PagedCache(k.half(), k.half(), one, one), lambda: PagedCache.empty(3, 16, 2, 64, torch.float8_e4m3fn, "cpu"),
                lambda: PagedCache.empty(3, 24, 2, 64, device="cpu"), lambda: PagedCache.empty(3, 16, 2, 96, device="cpu"),
                lambda: PagedCache.empty(0, 16, 2, 64, device="cpu"), lambda: PagedCache(k[0].half(), k[0].half()),
                lambda: PagedCache(*[torch.zeros((1, 16, 2, 64), dtype=torch.float8_e4m3fn)] * 2, one, one.double()),
                lambda: PagedCache(*[torch.zeros((1, 16, 2, 64), dtype=torch.float8_e4m3fn)] * 2, one[:1], one)):
        with pytest.raises(ValueError):
            bad()


def test_plain_attention_by_torch():
    """The plain form of the tests against torch's own, over a cache whose pages stand in any order."""
    gen = torch.Generator().manual_seed(1)
    kv = [torch.randn((5, 16, 2, 64), generator=gen).double() for _ in range(2)]
    q = torch.randn((4, 6, 64), generator=gen).to(torch.bfloat16)
    tables = torch.tensor([[4, 1, 2]])
    out, _, rows = paged.attention(q, kv, tables, [40], [1], [3], 0.125)
    assert rows.tolist() == [False, True, True, True]
    k, v = (t[tables[0]].reshape(48, 2, 64)[:40].permute(1, 0, 2).repeat_interleave(3, 0) for t in kv)
    mask = torch.arange(40)[None, :] <= torch.arange(37, 40)[:, None]
    want = torch.nn.functional.scaled_dot_product_attention(q[1:].double().permute(1, 0, 2), k, v, attn_mask=mask)
    assert torch.allclose(out[1:], want.permute(1, 0, 2))

def test_place():
    """Where the rows of a decoder's pass stand, and what does not fit."""
    s = S.Sequences(6, 3, 3, 4, 16, "cpu")
    s.place([[5, 2], [9]], [18, 2], [3, 2])
    assert s.slots.tolist() == [5 * 16 + 15, 32, 33, 144, 145, -1] and s.positions.tolist() == [15, 16, 17, 0, 1, 0]
    assert s.tables.tolist() == [[5, 2, -1, -1], [9, -1, -1, -1], [-1] * 4]
    assert s.lengths.tolist() == [18, 2, 0] and s.first.tolist() == [0, 3, 0] and s.n_new.tolist() == [3, 2, -1]
    for bad in (([[1]] * 4, [1] * 4, None), ([[1]], [17], [1]), ([[1]], [3], [4]), ([[1]], [2], [3]), ([[1, 2, 3, 4, 5]], [2], [1]),
                ([[1], [2], [3]], [3, 3, 3], [3, 3, 3]), ([[1]], [2, 3], None)):
        with pytest.raises(ValueError):
            s.place(*bad)
