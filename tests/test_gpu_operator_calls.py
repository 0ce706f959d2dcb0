"""GPU checks of calls of the adapters, the verification and the norms around a block that other tests do not make: views of one
buffer side by side, calls that would overwrite what they read."""
import pytest
import torch

from vllm_espalier import linear as LN
from vllm_espalier import workloads as WL
from vllm_espalier.adapters import Adapters

pytestmark = pytest.mark.gpu


def _store(K, outs, ranks, dtype, gen, dev, slots=None):
    store = Adapters(K, outs, slots=slots or len(ranks), max_rank=max(ranks), dtype=dtype, device=dev)
    for i, r in enumerate(ranks):
        store.load(i, [(torch.randn((r, K), generator=gen) * K ** -0.5).to(dtype) for _ in outs],
                   [(torch.randn((n, r), generator=gen) * r ** -0.5).to(dtype) for n in outs], 0.5)
    return store


@pytest.mark.parametrize("T", [1, 5, 300, 1200])
def test_lora_views_of_one_buffer(dev, T):
    """x, y and out side by side in the rows of one buffer are no overlap; x as y is one."""
    gen = torch.Generator().manual_seed(T)
    K = N = 64
    store = _store(K, [N], [8, 20], torch.bfloat16, gen, dev)
    wide = torch.randn((T, 3 * 64 + 4), generator=gen).to(torch.bfloat16).to(dev)
    before = wide.clone()
    rows = (torch.arange(T, dtype=torch.int32) % 3 - 1).to(dev)
    want = store.apply(before[:, :64].contiguous(), before[:, 64:128].contiguous(), rows)
    store.apply(wide[:, :64], wide[:, 64:128], rows, out=wide[:, 128:192])
    assert torch.equal(wide[:, 128:192].view(torch.int16), want.view(torch.int16))
    store.apply(wide[:, :64], wide[:, 64:128], rows)
    assert torch.equal(wide[:, 64:128].view(torch.int16), want.view(torch.int16))
    assert torch.equal(wide[:, :64], before[:, :64]) and torch.equal(wide[:, 192:], before[:, 192:])
    x = before[:, :64].contiguous()
    keep = x.clone()
    for y, out in ((x, None), (before[:, 64:128], x), (before[:, 60:124], before[:, 64:128])):
        with pytest.raises(RuntimeError, match="overlaps"):
            store.apply(x if y is x or out is x else wide[:, :64], y, rows, out=out)
    torch.cuda.synchronize()
    assert torch.equal(x, keep)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
def test_sandwich_of_no_rows(dev, ext, gate):
    rows = torch.empty((0, 64), dtype=torch.bfloat16, device=dev)
    w = torch.ones((64,), dtype=torch.bfloat16, device=dev)
    g = {"none": None, "channel": w, "token": rows[:, :1], "element": rows}[gate]
    out = torch.empty_like(rows)
    ext.sandwich_rmsnorm(rows, rows, rows, w, g, True, 0.5, w, 1e-6, rows, out)
    assert out.shape == (0, 64)


@pytest.mark.parametrize("T", [1, 9, 700])
def test_sandwich_in_place(dev, ext, T):
    """Either output in the place of h, a delta or a whole gate: the bits of outputs of their own."""
    gen = torch.Generator().manual_seed(T)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    tensors = {n: rnd(T, 520) for n in ("h", "d1", "d2", "gate")}
    post, pre = rnd(520), rnd(520)

    def run(ho, out):
        t = {n: v.clone() for n, v in tensors.items()}
        ho, out = (t[n] if n else torch.empty_like(t["h"]) for n in (ho, out))
        ext.sandwich_rmsnorm(t["h"], t["d1"], t["d2"], post, t["gate"], True, 0.5, pre, 1e-6, ho, out)
        return ho.view(torch.int16), out.view(torch.int16)

    want = run(None, None)
    for ho, out in (("h", None), ("h", "d1"), ("h", "d2"), ("h", "gate"), ("d1", "h"), ("gate", "d1"), ("d2", "gate")):
        assert all(torch.equal(w, g) for w, g in zip(want, run(ho, out))), (ho, out)
    h, d1 = tensors["h"].clone(), tensors["d1"]                # a row's gate that stands in the row itself
    for gate in (h[:, :1], h[:, 519:], h[:, 7:8]):
        alone = [torch.empty_like(h) for _ in range(2)]
        ext.sandwich_rmsnorm(tensors["h"], d1, None, post, gate.clone(), False, 0.5, pre, 1e-6, *alone)
        out = torch.empty_like(h)
        ext.sandwich_rmsnorm(h, d1, None, post, gate, False, 0.5, pre, 1e-6, h, out)
        assert all(torch.equal(g.view(torch.int16), w.view(torch.int16)) for g, w in zip((h, out), alone))
        h.copy_(tensors["h"])
    for ho, out in (("h", "h"), ("d1", "d1")):
        with pytest.raises(RuntimeError, match="overlap"):
            run(ho, out)
    if T == 1:
        return
    both = rnd(T + 1, 520)                                   # a row further
    with pytest.raises(RuntimeError, match="overlap"):
        ext.sandwich_rmsnorm(tensors["h"], both[1:], None, post, None, False, 1.0, pre, 1e-6, torch.empty_like(tensors["h"]), both[:T])


VIEWS = {"transposed": lambda rnd, T: rnd(256, T).t(), "every other column": lambda rnd, T: rnd(T, 512)[:, ::2],
         "odd stride": lambda rnd, T: rnd(T, 259)[:, :256], "odd start": lambda rnd, T: rnd(T * 256 + 1)[1:].view(T, 256),
         "expanded": lambda rnd, T: rnd(1, 256).expand(T, 256)}


@pytest.mark.parametrize("T", [1, 5, 1300])
@pytest.mark.parametrize("view", VIEWS)
def test_lora_rows_of_any_strides(dev, view, T):
    gen = torch.Generator().manual_seed(T)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    store = _store(256, [128, 16], [8, 20], torch.bfloat16, gen, dev)
    x, y = VIEWS[view](rnd, T), rnd(T, 144)
    rows = torch.stack([torch.randint(-1, 2, (T,), generator=gen), torch.full((T,), 7)], 1).to(torch.int32).to(dev)[:, 0]
    plain = x.clone(memory_format=torch.contiguous_format)
    want = store.apply(plain, y, rows.clone(memory_format=torch.contiguous_format), out=torch.empty_like(y))
    got = store.apply(x, y, rows, out=torch.empty_like(y))
    assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and (T < 5 or not torch.equal(got, y))


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("view", ["transposed", "every other column", "odd stride"])
def test_layer_rows_of_any_strides(dev, fused, view):
    """A layer takes the rows with adapters that it takes without."""
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    layer = LN.TrellisLinear([WL.matrix(256, 128, 4, "int6", torch.Generator(device=dev).manual_seed(1), dev)], 128, fused)
    store = layer.attach_adapters(2, 8)
    for i in range(2):
        store.load(i, [rnd(8, 256) / 16], [rnd(128, 8)], 0.5)
    x = VIEWS[view](rnd, 5)
    rows = torch.tensor([0, 9, 1, 9, -1, 9, 1, 9, 0, 9], dtype=torch.int32, device=dev)[::2]
    want = layer(x.contiguous(), rows.contiguous())
    assert torch.equal(layer(x, rows).view(torch.int16), want.view(torch.int16)) and not torch.equal(want, layer(x))


@pytest.mark.parametrize("fused", [True, False])
def test_layer_with_adapters_compiled(dev, fused):
    """espalier::add_adapters through torch.library's own checks, and a layer with adapters traced whole: the eager bits, with
    other rows and after a slot is loaded anew too."""
    gen = torch.Generator().manual_seed(7)
    rnd = lambda *s: torch.randn(s, generator=gen).to(torch.bfloat16).to(dev)  # noqa: E731
    mats = [WL.matrix(256, n, 4, "int6", torch.Generator(device=dev).manual_seed(n), dev) for n in (256, 128)]
    layer = LN.TrellisLinear(mats, 384, fused)
    store = layer.attach_adapters(2, 8)
    load = lambda i: store.load(i, [rnd(8, 256) / 16, None], [rnd(256, 8), None], 0.5)  # noqa: E731
    load(0), load(1)
    x, rows = rnd(5, 256), torch.tensor([0, -1, 1, 1, 0], dtype=torch.int32, device=dev)
    torch.library.opcheck(torch.ops.espalier.add_adapters.default,
                          (rnd(5, 384), x, rows, store.a, store.b, store.ranks, store.scales, store.out_features),
                          test_utils=("test_schema", "test_faketensor"))
    traced = torch.compile(layer, backend="aot_eager", fullgraph=True)
    for k in range(3):
        x, rows = rnd(5, 256), (rows + k) % 3 - 1
        with torch.no_grad():
            assert torch.equal(traced(x, rows).view(torch.int16), layer(x, rows).view(torch.int16)), k
        load(k % 2)


@pytest.mark.parametrize("T", [384, 700, 1151, 1152])
@pytest.mark.parametrize("slots", [16, 17, 40])
def test_lora_bits_whatever_the_slots(dev, T, slots):
    """As many slots as let the launches for many rows run, and more: the bits of short batches."""
    print(f"lora {T} rows, {slots} slots", flush=True)
    gen = torch.Generator().manual_seed(T)
    store = _store(512, [1024, 640], [16, 64, 40, 9] * 4, torch.bfloat16, gen, dev, slots=slots)
    x = torch.randn((T, 512), generator=gen).to(torch.bfloat16).to(dev)
    y = torch.randn((T, 1664), generator=gen).to(torch.bfloat16).to(dev)
    for rows in (torch.randint(-1, slots + 1, (T,), generator=gen), torch.arange(T) * 17 // T):
        rows = rows.to(torch.int32).to(dev)
        got = store.apply(x, y, rows, out=torch.full_like(y, float("nan")))
        short = torch.cat([store.apply(x[t:t + 90], y[t:t + 90].clone(), rows[t:t + 90]) for t in range(0, T, 90)])
        assert torch.equal(got.view(torch.int16), short.view(torch.int16))
