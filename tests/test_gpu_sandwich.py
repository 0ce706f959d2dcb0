"""GPU checks of sandwich_rmsnorm (csrc/sandwich.hip): the norms after and before a block with its gate and the residual scale,
against the formulas in 64 bits.

Bars, for every element: the residual within half a step of its type of the 64-bit value, plus 2^-16 of its terms (what the
fp32 arithmetic may lose: the sum of squares runs over at most 32 terms a lane and ten levels above it, 2^-18 together; a
sigmoid's exponent of up to 88 is off by 2^-24 of itself, 2^-17); the output likewise, from the residual as the kernel stored
it. Bit-equal to add_rmsnorm where the two coincide, and a row alone to the row in a batch.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _close(got, want, terms, dtype):
    got, want, terms = got.double().cpu(), want.cpu(), terms.cpu()
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -16 * terms + torch.finfo(dtype).smallest_normal * 2.0 ** -8
    bad = (got - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements off, by up to {float(((got - want).abs() / bound).max())} bounds"


def _inputs(T, D, dtype, deltas, post, gate, gen, dev):
    rnd = lambda *s, by=1.0: (torch.randn(s, generator=gen) * by).to(dtype).to(dev)  # noqa: E731
    g = None
    if gate == "element":
        g = rnd(T, D, by=2.0)
    elif gate == "channel":
        g = rnd(D)
    elif gate == "token":
        g = rnd(T, 1)
    elif gate == "view":                                     # the second half of a wider projection's rows
        g = rnd(T, 2 * D + 8)[:, D + 8:]
    return {"h": rnd(T, D, by=3.0), "d1": rnd(T, D), "d2": rnd(T, D, by=0.5) if deltas == 2 else None,
            "post": (1 + rnd(D, by=0.1).float()).to(dtype) if post else None, "pre": (1 + rnd(D, by=0.1).float()).to(dtype),
            "gate": g}


def _run(ext, i, sigmoid, scale, h_out=None, out=None, rows=slice(None)):
    cut = lambda t: None if t is None else t[rows].contiguous()  # noqa: E731
    gate = i["gate"]
    if gate is not None and gate.dim() == 2:
        gate = gate[rows]
    h = cut(i["h"])
    h_out = torch.full_like(h, float("nan")) if h_out is None else h_out
    out = torch.full_like(h, float("nan")) if out is None else out
    ext.sandwich_rmsnorm(h, cut(i["d1"]), cut(i["d2"]), i["post"], gate, sigmoid, scale, i["pre"], EPS, h_out, out)
    return h_out, out


def _check(i, sigmoid, scale, h_out, out, dtype):
    rms = lambda v, w: v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * (1.0 if w is None else w.double())  # noqa: E731
    u = i["d1"].double() + (0 if i["d2"] is None else i["d2"].double())
    size = i["d1"].double().abs() + (0 if i["d2"] is None else i["d2"].double().abs())
    if i["post"] is not None:
        inv = 1 / (u.square().mean(-1, keepdim=True) + EPS).sqrt()
        size = size * inv * i["post"].double().abs()
        u = rms(u, i["post"])
    f = 1.0
    if i["gate"] is not None:
        f = i["gate"].double()
        f = f.sigmoid() if sigmoid else f
    z = i["h"].double() + scale * f * u
    _close(h_out, z, i["h"].double().abs() + (scale * f * size).abs(), dtype)
    want = rms(h_out.double(), i["pre"])
    _close(out, want, want.abs(), dtype)


@pytest.mark.parametrize("T,D", [(1, 8), (1, 2048), (3, 520), (5, 1024), (2, 4096), (31, 2056), (1, 8192), (7, 8184), (300, 256),
                                 (600, 2048), (530, 5128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sandwich_sizes(dev, ext, T, D, dtype):
    print(f"sandwich {T} x {D} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(T * 8192 + D)
    i = _inputs(T, D, dtype, 2, True, "element", gen, dev)
    _check(i, True, 0.5, *_run(ext, i, True, 0.5), dtype)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "element", "view"])
@pytest.mark.parametrize("deltas,post", [(1, False), (1, True), (2, False), (2, True)])
@pytest.mark.parametrize("T", [4, 700])
def test_sandwich_forms(dev, ext, gate, deltas, post, T):
    gen = torch.Generator().manual_seed(deltas * 7 + post)
    i = _inputs(T, 640, torch.bfloat16, deltas, post, gate, gen, dev)
    for sigmoid in (False, True):
        _check(i, sigmoid, 0.22, *_run(ext, i, sigmoid, 0.22), torch.bfloat16)


@pytest.mark.parametrize("T,D", [(1, 2048), (9, 776), (1100, 2048), (520, 8192)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sandwich_equals_add_rmsnorm(dev, ext, T, D, dtype):
    """One delta, no gate, scale 1 and no norm behind the block: add_rmsnorm's bits, in place too."""
    gen = torch.Generator().manual_seed(D)
    i = _inputs(T, D, dtype, 1, False, "none", gen, dev)
    h, out = i["h"].clone(), torch.empty_like(i["h"])
    ext.add_rmsnorm(h, i["d1"], None, i["pre"], out, EPS)
    h2, out2 = _run(ext, i, False, 1.0)
    assert torch.equal(h.view(torch.int16), h2.view(torch.int16)) and torch.equal(out.view(torch.int16), out2.view(torch.int16))
    h3, out3 = i["h"].clone(), torch.empty_like(out)
    ext.sandwich_rmsnorm(h3, i["d1"], None, None, None, False, 1.0, i["pre"], EPS, h3, out3)
    assert torch.equal(h.view(torch.int16), h3.view(torch.int16)) and torch.equal(out.view(torch.int16), out3.view(torch.int16))


@pytest.mark.parametrize("D", [2048, 3640, 4096])
def test_sandwich_rows_alone_equal_batch(dev, ext, D):
    """Whatever the batch, a row has the bits that it has alone."""
    gen = torch.Generator().manual_seed(3)
    i = _inputs(1200, D, torch.bfloat16, 2, True, "element", gen, dev)
    h, out = _run(ext, i, True, 0.7)
    for n in (1, 33, 600):
        h1, out1 = _run(ext, i, True, 0.7, rows=slice(0, n))
        assert torch.equal(h1.view(torch.int16), h[:n].view(torch.int16)), n
        assert torch.equal(out1.view(torch.int16), out[:n].view(torch.int16)), n


def test_sandwich_odd_values(dev, ext):
    """A row of zeros stays finite, a row with a NaN or an infinity spoils itself alone, and gates far from zero close and
    open."""
    gen = torch.Generator().manual_seed(5)
    i = _inputs(6, 256, torch.bfloat16, 1, True, "element", gen, dev)
    i["d1"][0].zero_()
    i["h"][0].zero_()
    i["d1"][2, 7] = float("nan")
    i["d1"][4, 9] = float("inf")
    i["gate"][5] = -3e38
    i["gate"][3] = 3e38
    h, out = _run(ext, i, True, 1.0)
    ok = [0, 1, 3, 5]
    assert torch.isfinite(h[ok].float()).all() and torch.isfinite(out[ok].float()).all()
    assert int(out[0].abs().sum()) == 0
    assert torch.equal(h[5], i["h"][5])                      # a closed gate leaves the residual as it is
    assert not torch.isfinite(out[2].float()).any() and torch.isnan(h[4].float()).any()
    sub = {k: (v[ok] if torch.is_tensor(v) and v.dim() == 2 else v) for k, v in i.items()}
    sub["gate"] = sub["gate"].clamp(-80, 80)
    _check(sub, True, 1.0, h[ok], out[ok], torch.bfloat16)


def test_sandwich_graph_and_stream(dev, ext):
    gen = torch.Generator().manual_seed(6)
    i = _inputs(40, 2048, torch.bfloat16, 1, True, "token", gen, dev)
    h, out = torch.empty_like(i["h"]), torch.empty_like(i["h"])
    call = lambda: ext.sandwich_rmsnorm(i["h"], i["d1"], None, i["post"], i["gate"], True, 1.0, i["pre"], EPS, h, out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for k in range(3):
        i["d1"].copy_(torch.randn((40, 2048), generator=gen).to(torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        _check(i, True, 1.0, h, out, torch.bfloat16)


def test_sandwich_refusals(dev, ext):
    gen = torch.Generator().manual_seed(8)
    i = _inputs(4, 64, torch.bfloat16, 1, True, "element", gen, dev)
    ho, out = torch.empty_like(i["h"]), torch.empty_like(i["h"])

    def call(**over):
        a = dict(h=i["h"], d1=i["d1"], d2=None, post=i["post"], gate=i["gate"], pre=i["pre"], ho=ho, out=out)
        a.update(over)
        ext.sandwich_rmsnorm(a["h"], a["d1"], a["d2"], a["post"], a["gate"], False, 1.0, a["pre"], EPS, a["ho"], a["out"])

    call()
    for over in (dict(d1=i["d1"].float()), dict(d1=i["d1"][:3]), dict(post=i["post"][:32]), dict(pre=i["pre"].half()),
                 dict(gate=i["gate"][:, :32]), dict(gate=i["gate"][:3]), dict(gate=i["gate"].t().contiguous().t()),
                 dict(gate=torch.empty((4, 68), dtype=torch.bfloat16, device=dev)[:, 4:]), dict(out=out[:2]), dict(h=i["h"].cpu()),
                 dict(d1=i["d1"].cpu()), dict(ho=torch.empty((4, 128), dtype=torch.bfloat16, device=dev)[:, ::2])):
        with pytest.raises(RuntimeError):
            call(**over)
