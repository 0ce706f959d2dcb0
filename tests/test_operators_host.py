"""Refusals of the adapters, the verification and the norms around a block, on the CPU: the C ABI's argument checks fail with a
code and a message before any HIP call, and an Adapters store checks what is loaded into it."""
import ctypes
from pathlib import Path

import pytest
import torch

from vllm_espalier.adapters import Adapters

LIB = Path(__file__).resolve().parent.parent / "vllm-espalier_amd" / "vllm_espalier" / "libespalier_hip.so"
P, I64, INT, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double


@pytest.fixture(scope="module")
def lib(ext):
    L = ctypes.CDLL(str(LIB))
    L.esp_last_error.restype = ctypes.c_char_p
    L.esp_sandwich_rmsnorm.argtypes = [P, P, P, P, P, I64, I64, INT, F64, P, P, P, I64, I64, F64, INT, P]
    L.esp_lora.argtypes = [P, I64, P, I64, P, I64, P, I64, I64, I64, ctypes.POINTER(I64), P, P, P, P, I64, I64, INT, P, I64, P]
    L.esp_lora_scratch.argtypes, L.esp_lora_scratch.restype = [I64] * 4, I64
    L.esp_verify.argtypes = [P, INT, I64, I64, I64, P, P, P, I64, I64, P, P, I64, P, P, I64, I64, P, P, P, P, I64, P]
    L.esp_verify_scratch.argtypes, L.esp_verify_scratch.restype = [I64, I64, I64], I64
    return L


def _sandwich(lib, **over):
    a = dict(h=16, d1=16, d2=None, post=16, gate=16, row=64, col=1, pre=16, ho=16, out=16, T=4, D=64, dtype=1)
    a.update(over)
    return lib.esp_sandwich_rmsnorm(a["h"], a["d1"], a["d2"], a["post"], a["gate"], a["row"], a["col"], 0, 1.0, a["pre"],
                                    a["ho"], a["out"], a["T"], a["D"], 1e-6, a["dtype"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(h=None), "null"), (dict(d1=None), "null"), (dict(pre=None), "null"), (dict(ho=None), "null"), (dict(dtype=2), "bf16"),
    (dict(D=0), "multiple of 8"), (dict(D=12), "multiple of 8"), (dict(D=8200), "at most"), (dict(T=1 << 31), "rows"),
    (dict(d2=8), "aligned"), (dict(post=24), "aligned"), (dict(gate=24), "gate"), (dict(row=-64), "stride"),
    (dict(row=60), "gate"), (dict(col=2), "stride"), (dict(col=0, gate=17), "gate")])
def test_sandwich_argument_errors(lib, over, needle):
    assert _sandwich(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def test_no_rows_is_no_call(lib):
    assert _sandwich(lib, T=0) == 0
    assert _lora(lib, T=0, x=None, y=None) == 0
    assert _verify(lib, B=0, logits=None) == 0


def _lora(lib, **over):
    a = dict(x=16, xs=64, y=16, ys=32, out=16, os=32, rows=16, T=4, K=64, S=1, cols=[32], A=16, B=16, ranks=16, scales=16,
             slots=2, R=16, dtype=1, scratch=16, numel=1 << 40)
    a.update(over)
    cols = (I64 * len(a["cols"]))(*a["cols"])
    return lib.esp_lora(a["x"], a["xs"], a["y"], a["ys"], a["out"], a["os"], a["rows"], a["T"], a["K"], a["S"], cols, a["A"],
                        a["B"], a["ranks"], a["scales"], a["slots"], a["R"], a["dtype"], a["scratch"], a["numel"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(dtype=2), "bf16"), (dict(T=-1), "rows"), (dict(T=1 << 24), "rows"), (dict(S=0), "matrices"),
    (dict(S=5, cols=[16] * 5), "matrices"), (dict(K=72), "multiple of 16"), (dict(K=0), "multiple of 16"),
    (dict(T=(1 << 24) - 1, cols=[8192]), "blocks of 64 rows"),
    (dict(R=8), "multiple of 16"), (dict(R=272), "at most"), (dict(slots=0), "adapters"), (dict(cols=[24]), "columns"),
    (dict(cols=[0]), "columns"), (dict(x=None), "null"), (dict(scratch=None), "null"), (dict(ranks=None), "null"),
    (dict(xs=32), "overlap"), (dict(ys=16), "overlap"), (dict(os=36), "in place"), (dict(x=20), "aligned"),
    (dict(xs=66), "aligned"), (dict(out=24, os=34), "aligned"), (dict(A=24), "aligned"), (dict(scratch=20), "aligned"),
    (dict(numel=63), "scratch")])
def test_lora_argument_errors(lib, over, needle):
    assert _lora(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def test_scratch_sizes(lib):
    assert lib.esp_lora_scratch(4, 64, 1, 16) >= 64
    assert lib.esp_lora_scratch(0, 64, 1, 16) == 0
    assert lib.esp_verify_scratch(4, 2, 100) > 0
    assert lib.esp_verify_scratch(0, 2, 100) == 0


def _verify(lib, **over):
    a = dict(logits=16, dtype=1, stride=64, R=8, V=64, first=16, n=16, drafts=16, B=2, G=3, uniform=16, race=16, rs=64, temp=16,
             probs=None, pb=192, pr=64, tokens=16, counts=16, lp=16, scratch=16, bytes=1 << 30)
    a.update(over)
    return lib.esp_verify(a["logits"], a["dtype"], a["stride"], a["R"], a["V"], a["first"], a["n"], a["drafts"], a["B"], a["G"],
                          a["uniform"], a["race"], a["rs"], a["temp"], a["probs"], a["pb"], a["pr"], a["tokens"], a["counts"],
                          a["lp"], a["scratch"], a["bytes"], None)


@pytest.mark.parametrize("over,needle", [
    (dict(dtype=3), "dtype"), (dict(B=-1), "requests"), (dict(B=1 << 21), "requests"), (dict(B=1 << 20, V=1 << 24, stride=1 << 24, rs=1 << 24, G=1024), "blocks"), (dict(G=-1), "drafts"),
    (dict(G=1025), "drafts"), (dict(R=1 << 31), "rows"), (dict(V=0), "V"), (dict(V=1 << 28), "V"), (dict(logits=None), "null"),
    (dict(first=None), "null"), (dict(drafts=None), "null"), (dict(race=None), "null"), (dict(scratch=None), "null"),
    (dict(stride=63), "overlap"), (dict(rs=63), "overlap"), (dict(pr=-1), "stride"), (dict(logits=17), "aligned"),
    (dict(logits=18, dtype=2), "aligned"), (dict(scratch=24), "scratch"), (dict(bytes=100), "scratch")])
def test_verify_argument_errors(lib, over, needle):
    assert _verify(lib, **over) == 1
    assert needle in lib.esp_last_error().decode()


def test_adapters_layout():
    """The places of the elements in a slot, as the C header gives them."""
    gen = torch.Generator().manual_seed(1)
    K, outs, r = 48, [144, 16], 19
    store = Adapters(K, outs, slots=1, max_rank=20, device="cpu")
    a = [torch.randn((r, K), generator=gen).to(torch.bfloat16) for _ in outs]
    b = [torch.randn((n, r), generator=gen).to(torch.bfloat16) for n in outs]
    store.load(0, a, b)
    for s, first in ((0, 0), (1, 2)):
        for j, k in ((0, 0), (18, 47), (7, 33), (16, 12)):
            assert store.a[0, s, j // 16, k // 32, k % 32 // 8, j % 16, k % 8] == a[s][j, k]
        for n, j in ((0, 0), (outs[s] - 1, 18), (13, 9), (outs[s] // 2, 17)):
            assert store.b[0, first + n // 128, j // 16, n % 8, j % 16 // 8, n % 128 // 8, j % 8] == b[s][n, j]
    assert int((store.a != 0).sum()) == sum(int((t != 0).sum()) for t in a)
    assert int((store.b != 0).sum()) == sum(int((t != 0).sum()) for t in b)


def test_adapters_checks():
    for bad in (dict(in_features=24), dict(out_features=[16, 8]), dict(out_features=[]), dict(out_features=[16] * 5), dict(slots=0),
                dict(max_rank=0), dict(max_rank=257), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            Adapters(**{**dict(in_features=32, out_features=[16, 32], slots=2, max_rank=8, device="cpu"), **bad})
    store = Adapters(32, [16, 32], slots=2, max_rank=8, device="cpu")
    assert store.a.shape == (2, 2, 1, 1, 4, 16, 8) and store.b.shape == (2, 2, 1, 8, 2, 16, 8)
    a, b = [torch.ones((4, 32)), None], [torch.ones((16, 4)), None]
    store.load(1, a, b, scale=0.5)
    assert store.ranks.tolist() == [[0, 0], [4, 0]] and store.scales[1, 0] == 0.5
    assert float(store.a[1, 0].float().sum()) == 128 and float(store.b[1, 0].float().sum()) == 64
    assert not store.a[1, 1].any() and not store.b[1, 1].any()
    bad_b = [torch.ones((16, 5)), None]
    for args in ((2, a, b), (-1, a, b), (0, a[:1], b), (0, a, [b[0], torch.ones((32, 4))]), (0, a, bad_b),
                 (0, [torch.ones((9, 32)), None], [torch.ones((16, 9)), None]), (0, [torch.ones((4, 16)), None], b),
                 (0, [torch.ones((0, 32)), None], [torch.ones((16, 0)), None])):
        with pytest.raises(ValueError):
            store.load(*args)
    assert store.ranks.tolist() == [[0, 0], [4, 0]]          # a refused adapter leaves the slots as they were
    with pytest.raises(ValueError):
        store.load(1, [torch.ones((4, 32)), a[0]], bad_b)
    assert store.ranks.tolist() == [[0, 0], [4, 0]]
    store.clear(1)
    assert int(store.ranks.sum()) == 0
