"""Calls of the adapters, the verification and the norms around a block that have to be refused, or must leave nothing behind, on
the CPU: the package's own checks in front of the extension, and the C ABI's before any HIP call."""
import ctypes
import gc
import weakref
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_espalier import linear as LN
from vllm_espalier import ops  # noqa: F401  (registers the espalier::* ops)
from vllm_espalier import workloads as WL
from vllm_espalier.adapters import Adapters

LIB = Path(__file__).resolve().parent.parent / "vllm-espalier_amd" / "vllm_espalier" / "libespalier_hip.so"
P, I64, INT, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double


@pytest.fixture(scope="module")
def lib(ext):
    L = ctypes.CDLL(str(LIB))
    L.esp_last_error.restype = ctypes.c_char_p
    L.esp_lora.argtypes = [P, I64, P, I64, P, I64, P, I64, I64, I64, ctypes.POINTER(I64), P, P, P, P, I64, I64, INT, P, I64, P]
    L.esp_lora_scratch.argtypes, L.esp_lora_scratch.restype = [I64] * 4, I64
    L.esp_sandwich_rmsnorm.argtypes = [P, P, P, P, P, I64, I64, INT, F64, P, P, P, I64, I64, F64, INT, P]
    return L


def _layer(monkeypatch, in_features, outs):
    """A TrellisLinear on the CPU whose coded matrices give zeros."""
    layer = LN.TrellisLinear([], sum(outs), False)
    monkeypatch.setattr(layer, "_base", lambda x: torch.zeros((*x.shape[:-1], sum(outs)), dtype=x.dtype))
    layer.adapters = Adapters(in_features, outs, slots=1, max_rank=4, device="cpu")
    return layer


@pytest.mark.parametrize("have,given", [(64, 48), (48, 64), (32, 16), (16, 32), (64, 96)])
def test_rows_of_another_width_refused(monkeypatch, have, given):
    """Widths that differ inside a unit of 32 k too, which the shape of the padded A does not tell apart."""
    store = Adapters(have, [32], slots=1, max_rank=4, device="cpu")
    x, y = torch.zeros((3, given), dtype=torch.bfloat16), torch.zeros((3, 32), dtype=torch.bfloat16)
    rows = torch.zeros((3,), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="in_features"):
        store.apply(x, y, rows)
    with pytest.raises(RuntimeError, match="in_features"):
        store.apply(x[0], y, rows)
    with pytest.raises(RuntimeError, match="in_features"):
        _layer(monkeypatch, have, [32])(x.view(1, 3, given), rows)
    with pytest.raises(RuntimeError, match="in_features"):
        torch.ops.espalier.add_adapters(y, x, rows, store.a, store.b, store.ranks, store.scales, store.out_features, have)


@pytest.mark.parametrize("x,xs,y,ys,out,os,needle", [
    (4096, 64, 4096, 64, 4096, 64, "overlaps x"),            # y = x, in place: rows that other workgroups still read
    (4096, 64, 65536, 64, 4096, 64, "overlaps x"),           # out = x
    (4096, 64, 65536, 64, 4096 + 3 * 128 + 64, 64, "overlaps x"),        # the last row alone
    (4096, 128, 65536, 128, 4096 + 96, 128, "overlaps x"),   # side by side in one buffer, but for 16 columns
    (4096, 128, 65536, 128, 4096 - 96, 128, "overlaps x"),
    (4096, 100, 65536, 64, 4096 + 2 * 136, 68, "overlaps x"),      # different strides
    (65536, 64, 4096, 64, 4096 + 128, 64, "overlaps y"),     # a row further
    (65536, 64, 4096, 128, 4096 + 32, 128, "overlaps y"),
    (65536, 64, 4096, 128, 4096 + 64, 68, "overlaps y")])
def test_lora_overlap_refused(lib, x, xs, y, ys, out, os, needle):
    """4 rows of 64 -> 64 in 16-bit elements at made-up addresses: refused before anything reads them."""
    rc = lib.esp_lora(x, xs, y, ys, out, os, 16, 4, 64, 1, (I64 * 1)(64), 16, 16, 16, 16, 1, 16, 1, 16, 1 << 20, None)
    assert rc == 1 and needle in lib.esp_last_error().decode()
    one = lib.esp_lora(x, xs, y, ys, x, os, 16, 1, 64, 1, (I64 * 1)(64), 16, 16, 16, 16, 1, 16, 1, 16, 1 << 20, None)
    assert one == 1 and "overlaps x" in lib.esp_last_error().decode()


def test_sandwich_of_no_rows(lib):
    """A batch of no rows, whose tensors have no address, is no error; what does not fit is one even so."""
    none = lambda D, dtype=1: lib.esp_sandwich_rmsnorm(None, None, None, 16, None, 0, 0, 0, 1.0, 16, None, None, 0, D, 1e-6,  # noqa: E731
                                                       dtype, None)
    assert none(64) == 0
    assert none(12) == 1 and none(64, 2) == 1


FAR = 1 << 20                                                # 4 rows of 64 elements of 16 bits: 512 bytes a tensor


@pytest.mark.parametrize("over,needle", [
    (dict(out=0), "two outputs"), (dict(out=2 * FAR, ho=2 * FAR + 256), "two outputs"),
    (dict(ho=128), "other rows"), (dict(out=FAR + 128), "other rows"), (dict(out=3 * FAR - 128), "other rows"),
    (dict(out=4 * FAR - 384), "weight"), (dict(ho=5 * FAR), "weight"), (dict(out=6 * FAR), "gate"),
    (dict(out=6 * FAR, row=128, col=0), "gate"), (dict(ho=6 * FAR + 256, row=64, col=0), "gate"),
    (dict(out=6 * FAR + 128, row=64), "gate"), (dict(ho=6 * FAR, row=72), "gate")])
def test_sandwich_overlap_refused(lib, over, needle):
    """An output over another one, another row of an input, a weight, or a gate that other workgroups read: refused."""
    a = dict(ho=0, out=7 * FAR, row=0, col=1)                # h_out = h; h, d1, d2, the weights and the gate far apart
    a.update(over)
    at = lambda n: FAR + n  # noqa: E731
    rc = lib.esp_sandwich_rmsnorm(at(0), at(FAR), at(3 * FAR), at(4 * FAR), at(6 * FAR), a["row"], a["col"], 0, 1.0, at(5 * FAR),
                                  at(a["ho"]), at(a["out"]), 4, 64, 1e-6, 1, None)
    assert rc == 1 and needle in lib.esp_last_error().decode()


def test_loaded_parameters_leave_no_graph():
    """Parameters that require grad, loaded with grad mode on: the store's tensors stay plain, and hold none of what was loaded."""
    store = Adapters(32, [16, 32], slots=2, max_rank=8, device="cpu")
    kept = []
    for k in range(2):
        a = [torch.nn.Parameter(torch.randn((4, 32))) for _ in range(2)]
        b = [torch.nn.Parameter(torch.randn((n, 4))) for n in (16, 32)]
        store.load(k, a, [p * 2 for p in b])
        kept += [weakref.ref(p) for p in a + b]
        assert torch.equal(store.a[k, 1, 0, 0, :, :4].transpose(0, 1).reshape(4, 32), a[1].detach().to(torch.bfloat16))
    store.clear(0)
    for t in (store.a, store.b, store.ranks, store.scales):
        assert not t.requires_grad and t.grad_fn is None
    del a, b
    gc.collect()
    assert not any(r() is not None for r in kept)


def test_adapters_move_with_their_layer():
    """To another device (that of no data here) with the layer's buffers, before the adapters are attached or after; a change of
    dtype, which is no move, leaves them as they are."""
    gen = torch.Generator().manual_seed(1)
    mats = [WL.matrix(128, n, 4, "int6", gen, torch.device("cpu")) for n in (128, 256)]
    layer = LN.TrellisLinear(mats, 384, False)
    store = layer.attach_adapters(2, 8, torch.float16)
    a, scales = store.a, store.scales
    layer.float()
    layer.to("cpu")
    assert store.a is a and store.scales is scales and store.a.dtype == torch.float16 and store.scales.dtype == torch.float32
    outer = torch.nn.Sequential(layer).to("meta")
    assert outer[0].adapters is store and layer.trellis_0.device.type == "meta"
    for t in (store.a, store.b, store.ranks, store.scales):
        assert t.device.type == "meta"
    assert layer.attach_adapters(2, 8).a.device.type == "meta"


def test_add_adapters_fake_form():
    """Under fake tensors the op gives nothing, reaches no extension, and is known to change y alone."""
    with FakeTensorMode():
        store = Adapters(64, [32], slots=1, max_rank=4, device="cpu")
        y = torch.empty((3, 32), dtype=torch.bfloat16)
        got = torch.ops.espalier.add_adapters(y, torch.empty((3, 64), dtype=torch.bfloat16), torch.empty((3,), dtype=torch.int32),
                                              store.a, store.b, store.ranks, store.scales, store.out_features)
    assert got is None
    args = torch.ops.espalier.add_adapters.default._schema.arguments
    assert [a.name for a in args if a.alias_info is not None and a.alias_info.is_write] == ["y"]


@pytest.mark.parametrize("T", [1, 16, 383, 384, 512, 1000, 1151, 1152, 4096])
@pytest.mark.parametrize("N,S,R", [(5120, 3, 64), (2048, 1, 128), (64, 1, 16)])
def test_lora_scratch_of_either_launches(lib, T, N, S, R):
    """The size does not know the slots, which choose between the launches for few and for many rows below 1152: it covers the four
    sums of 16 x 16 that the few keep a rank tile and 16 rows, and from there on the many's operands and exponents."""
    tiles = -(-T // 16) * S * (R // 16)
    assert lib.esp_lora_scratch(T, N, S, R) >= tiles * (4 * 256 if T < 1152 else 256 + 16)
