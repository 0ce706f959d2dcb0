"""GPU checks of the adapters (csrc/lora.hip, vllm_espalier/adapters.py) against the products in 64 bits.

The bar of every element, derived: half a step of the output's type, plus what 32 bits lose on the way. A sum of K products is
off by at most K 2^-24 of the sum of their magnitudes; its 16-bit high part and rest are together off by 2^-16 (bf16), or, in
fp16, by 2^-20 of the largest of the row's t; r more products by r 2^-24; the last addition by 2^-24 of its terms.
Rows without an adapter keep their bits, and a row alone has those that it has in any batch.
"""
import pytest
import torch

from vllm_espalier import dense as Dn
from vllm_espalier import workloads as WL
from vllm_espalier.adapters import Adapters

pytestmark = pytest.mark.gpu


def _store(K, outs, ranks, dtype, gen, dev, max_rank=None, skip=()):
    """A store with one adapter a rank, and its matrices on the CPU; `skip`: (slot, matrix) left alone."""
    store = Adapters(K, outs, slots=len(ranks), max_rank=max_rank or max(ranks), dtype=dtype, device=dev)
    a, b, scales = [], [], []
    for i, r in enumerate(ranks):
        low = [None if (i, s) in skip else (torch.randn((r, K), generator=gen) * K ** -0.5).to(dtype) for s in range(len(outs))]
        high = [None if (i, s) in skip else (torch.randn((n, r), generator=gen) * r ** -0.5).to(dtype) for s, n in enumerate(outs)]
        a.append(low), b.append(high), scales.append(0.5 + i % 3)
        store.load(i, low, high, scale=scales[-1])
    return store, a, b, scales


def _want(x, y, rows, a, b, scales, outs, dtype):
    """(out, bound) in 64 bits."""
    x, out = x.cpu().double(), y.cpu().double()[:, :sum(outs)].clone()
    bound = torch.zeros_like(out)
    K = x.shape[1]
    for t, who in enumerate(rows.tolist()):
        if not 0 <= who < len(a):
            continue
        col = 0
        for low, high, n in zip(a[who], b[who], outs):
            cols = slice(col, col + n)
            col += n
            if low is None:
                continue
            r = low.shape[0]
            low, high = low.double(), high.double()
            v = scales[who] * (low @ x[t])
            size = scales[who] * (low.abs() @ x[t].abs())
            off = K * 2.0 ** -24 * size + (2.0 ** -16 * v.abs() if dtype == torch.bfloat16 else 2.0 ** -20 * v.abs().max())
            delta = high @ v
            bound[t, cols] = high.abs() @ (off + r * 2.0 ** -24 * v.abs()) + 2.0 ** -24 * (out[t, cols].abs() + delta.abs())
            out[t, cols] += delta
    return out, bound + torch.finfo(dtype).eps / 2 * out.abs() + torch.finfo(dtype).smallest_normal * 2.0 ** -8


def _check(got, x, y, rows, a, b, scales, outs, dtype):
    want, bound = _want(x, y, rows, a, b, scales, outs, dtype)
    N = sum(outs)
    off = (got.cpu().double()[:, :N] - want).abs()
    assert not (off > bound).any(), f"{int((off > bound).sum())} elements off, by up to {float((off / bound).max())} bounds"
    none = [t for t, who in enumerate(rows.tolist()) if not 0 <= who < len(a)]
    assert torch.equal(got[none, :N].view(torch.int16).cpu(), y[none, :N].view(torch.int16).cpu())


def _rows(T, L, gen, mixed=True):
    rows = torch.randint(-1, L, (T,), generator=gen) if mixed else torch.arange(T) * L // T
    return rows.to(torch.int32)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 256, 257, 530, 1601])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora_rows(dev, T, dtype):
    print(f"lora rows {T} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(T)
    K, outs = 528, [64, 16, 48]
    store, a, b, scales = _store(K, outs, [16, 3, 40, 8, 17], dtype, gen, dev, skip={(1, 0), (4, 2)})
    x = torch.randn((T, K), generator=gen).to(dtype).to(dev)
    y = torch.randn((T, sum(outs)), generator=gen).to(dtype).to(dev)
    for rows in (_rows(T, 5, gen), _rows(T, 5, gen, mixed=False)):
        out = torch.full_like(y, float("nan"))
        assert store.apply(x, y, rows.to(dev), out=out) is out
        _check(out, x, y, rows, a, b, scales, outs, dtype)
        inplace = y.clone()
        assert store.apply(x, inplace, rows.to(dev)) is inplace
        assert torch.equal(inplace.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("K,outs,ranks", [
    (16, [16], [1]), (64, [64], [16, 16]), (80, [16, 16, 16, 16], [2, 5]), (2048, [4096, 512, 512], [16, 64]), (4096, [2048], [8]),
    (512, [2048], [256, 31]), (1040, [80, 1024], [128, 1]), (5120, [32], [33]), (2048, [64] * 4, [64, 48]), (96, [8208], [12])])
@pytest.mark.parametrize("T", [3, 40, 300, 1537])
def test_lora_shapes(dev, K, outs, ranks, T):
    print(f"lora {K} -> {outs}, ranks {ranks}, {T} rows", flush=True)
    gen = torch.Generator().manual_seed(K + T)
    dtype = torch.bfloat16 if T != 40 else torch.float16
    store, a, b, scales = _store(K, outs, ranks, dtype, gen, dev)
    x = torch.randn((T, K), generator=gen).to(dtype).to(dev)
    y = torch.randn((T, sum(outs)), generator=gen).to(dtype).to(dev)
    rows = _rows(T, len(ranks), gen)
    _check(store.apply(x, y, rows.to(dev), out=torch.empty_like(y)), x, y, rows, a, b, scales, outs, dtype)


@pytest.mark.parametrize("T", [5, 300, 1700])
def test_lora_rows_alone_equal_batch(dev, T):
    """A row's bits are its own: alone, in windows and in the whole batch, whatever stands beside it."""
    gen = torch.Generator().manual_seed(2)
    K, outs = 2048, [512, 256]
    store, *_ = _store(K, outs, [16, 64, 9], torch.bfloat16, gen, dev)
    x = torch.randn((T, K), generator=gen).to(torch.bfloat16).to(dev)
    y = torch.randn((T, sum(outs)), generator=gen).to(torch.bfloat16).to(dev)
    rows = _rows(T, 3, gen).to(dev)
    whole = store.apply(x, y, rows, out=torch.empty_like(y))
    for step in (1, 7, 64, 290, 1543):
        for r0 in range(0, T, step * (1 if step > 1 else 37) * (1 + T // 600)):
            part = slice(r0, r0 + step)
            got = store.apply(x[part], y[part], rows[part], out=torch.empty_like(y[part]))
            assert torch.equal(got.view(torch.int16), whole[part].view(torch.int16)), (step, r0)


@pytest.mark.parametrize("T", [6, 290, 1540])
def test_lora_strides_and_columns(dev, T):
    """Views of wider buffers, whose rows are 8-byte aligned only, a padded output, and rows of no or a far adapter."""
    gen = torch.Generator().manual_seed(4)
    K, outs, dtype = 192, [48, 32], torch.bfloat16
    store, a, b, scales = _store(K, outs, [16, 20], dtype, gen, dev)
    wide = torch.randn((T, K + 20), generator=gen).to(dtype).to(dev)
    x = wide[:, 4:4 + K]
    pad = torch.randn((T, 100), generator=gen).to(dtype).to(dev)
    y = pad[:, 4:]                                           # 80 columns of the layer and 16 more, rows of 100
    before = pad.clone()
    rows = torch.tensor([0, 1, -1, 2, 2 ** 31 - 1, -2 ** 31] * -(-T // 6), dtype=torch.int32)[:T]
    store.apply(x, y, rows.to(dev))
    _check(y, x, before[:, 4:], rows, a, b, scales, outs, dtype)
    assert torch.equal(pad[:, :4], before[:, :4]) and torch.equal(pad[:, 84:], before[:, 84:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [4, 272, 1552])
def test_lora_isolation(dev, T, dtype):
    """What is not a row's own does not reach it: NaN behind a slot's rank, infinities in another adapter, a NaN in another
    row's input; an adapter cleared, loaded again with a smaller rank, or without one of its matrices."""
    gen = torch.Generator().manual_seed(9)
    K, outs = 256, [64, 32]
    store, a, b, scales = _store(K, outs, [5, 24, 16], dtype, gen, dev, max_rank=32)
    for i, r in enumerate([5, 24, 16]):                      # tiles of 16 ranks past the adapter's
        store.a[i, :, -(-r // 16):] = float("nan")
        store.b[i, :, -(-r // 16):] = float("nan")
    store.a[2], store.b[2] = float("inf"), float("nan")
    x = torch.randn((T, K), generator=gen).to(dtype).to(dev)
    y = torch.randn((T, sum(outs)), generator=gen).to(dtype).to(dev)
    rows = torch.tensor([0, 2, 1, -1] * (T // 4), dtype=torch.int32)
    x[1] = float("nan")
    x[3] = float("nan")                                      # of a row without an adapter
    out = store.apply(x, y, rows.to(dev), out=torch.empty_like(y))
    clean = [t for t in range(T) if t % 4 != 1]
    _check(out[clean], x[clean], y[clean], rows[clean], a[:2], b[:2], scales, outs, dtype)
    low = [None, (torch.randn((2, K), generator=gen) / 16).to(dtype)]
    high = [None, torch.randn((32, 2), generator=gen).to(dtype)]
    store.load(2, low, high, scale=3.0)
    store.clear(1)
    x[1] = x[0]
    got = store.apply(x, y, rows.to(dev), out=torch.empty_like(y))
    rows2 = torch.where(rows == 1, -1, rows)
    _check(got, x.nan_to_num(), y, rows2, [a[0], None, low], [b[0], None, high], [scales[0], 1.0, 3.0], outs, dtype)


@pytest.mark.parametrize("size", [1e-6, 1.0, 3e3])
def test_lora_fp16_range(dev, size):
    """fp16 rows whose t is far below or above fp16's own range keep 32-bit precision between the products."""
    gen = torch.Generator().manual_seed(12)
    K, outs, dtype, T = 512, [64], torch.float16, 20
    store = Adapters(K, outs, slots=2, max_rank=16, dtype=dtype, device=dev)
    a = [[(torch.randn((16, K), generator=gen) * 2.0 ** -4).to(dtype)] for _ in range(2)]
    b = [[(torch.randn((64, 16), generator=gen) * 2.0 ** -7).to(dtype)] for _ in range(2)]
    scales = [size, size / 2]
    for i in range(2):
        store.load(i, a[i], b[i], scale=scales[i])
    x = (torch.randn((T, K), generator=gen) * (20 if size > 1 else 1)).to(dtype).to(dev)
    y = (torch.randn((T, 64), generator=gen) * min(size, 1.0)).to(dtype).to(dev)
    rows = _rows(T, 2, gen)
    scales = [float(torch.tensor(s)) for s in scales]
    _check(store.apply(x, y, rows.to(dev), out=torch.empty_like(y)), x, y, rows, a, b, scales, outs, dtype)


@pytest.mark.parametrize("T,ranks", [(3, [8, 8]), (20, [8, 40]), (1600, [16, 64])])
def test_lora_untouched_bits(dev, T, ranks):
    """Matrices without ranks, cleared slots and rows without adapters: y's bits, zeros of both signs and NaN among them, in place
    and not; the other matrix of the same adapter as ever."""
    gen = torch.Generator().manual_seed(19)
    K, outs, dtype = 128, [48, 80], torch.bfloat16
    store, a, b, scales = _store(K, outs, ranks, dtype, gen, dev, skip={(0, 1)})
    store.clear(1)
    x = torch.randn((T, K), generator=gen).to(dtype).to(dev)
    y = torch.randn((T, 128), generator=gen).to(dtype)
    y[:, ::3] = -0.0
    y[:, 60] = float("nan")
    y = y.to(dev)
    rows = torch.tensor([0, 1, -1] * -(-T // 3), dtype=torch.int32)[:T]
    for out in (torch.zeros_like(y), y.clone()):
        got = store.apply(x, y if out.any() == 0 else out, rows.to(dev), out=out)
        assert torch.equal(got[:, 48:].view(torch.int16), y[:, 48:].view(torch.int16))
        bare = rows != 0
        assert torch.equal(got[bare.to(dev)].view(torch.int16), y[bare.to(dev)].view(torch.int16))
        _check(got[:, :48], x, y[:, :48], torch.where(rows == 0, 0, -1), [a[0][:1]], [b[0][:1]], scales, outs[:1], dtype)


def test_lora_prompt_in_a_graph(dev):
    """The launches for many rows captured, and replayed with other rows and inputs."""
    gen = torch.Generator().manual_seed(23)
    K, outs, T = 256, [256, 128], 1700
    store, a, b, scales = _store(K, outs, [16, 70], torch.bfloat16, gen, dev)
    x = torch.randn((T, K), generator=gen).to(torch.bfloat16).to(dev)
    y = torch.randn((T, 384), generator=gen).to(torch.bfloat16).to(dev)
    rows, out = torch.zeros((T,), dtype=torch.int32, device=dev), torch.empty_like(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        store.apply(x, y, rows, out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        store.apply(x, y, rows, out=out)
    for k in range(3):
        rows.copy_(_rows(T, 2, gen, mixed=k == 1))
        x.copy_(torch.randn((T, K), generator=gen).to(torch.bfloat16))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        eager = store.apply(x, y, rows, out=torch.empty_like(y))
        assert torch.equal(eager.view(torch.int16), out.view(torch.int16)), k
    _check(out, x, y, rows.cpu(), a, b, scales, outs, torch.bfloat16)


def test_lora_long_rows_and_many_columns(dev):
    """Long K with few and many rows (x in several parts a run), and more columns than the one launch takes."""
    gen = torch.Generator().manual_seed(27)
    for K, outs, ranks, T in ((10256, [64], [16, 33], 9), (10256, [64], [16, 33], 1590), (64, [40000], [16], 16), (6160, [128], [4], 16)):
        print(f"lora {K} -> {outs}, {T} rows", flush=True)
        store, a, b, scales = _store(K, outs, ranks, torch.bfloat16, gen, dev)
        x = torch.randn((T, K), generator=gen).to(torch.bfloat16).to(dev)
        y = torch.randn((T, sum(outs)), generator=gen).to(torch.bfloat16).to(dev)
        rows = _rows(T, len(ranks), gen)
        out = store.apply(x, y, rows.to(dev), out=torch.empty_like(y))
        some = torch.arange(0, T, max(1, T // 40))
        _check(out[some], x[some], y[some], rows[some], a, b, scales, outs, torch.bfloat16)


@pytest.mark.parametrize("K", [16, 96, 1040, 2048, 2064, 4096, 4112, 8192, 8208])
@pytest.mark.parametrize("ranks,dtype", [([5, 16], torch.bfloat16), ([96, 16, 40, 33, 81], torch.bfloat16),
                                         ([96, 16, 40, 33, 81], torch.float16)])
@pytest.mark.parametrize("mixed", [False, True])
def test_lora_prompt_tiles(dev, K, ranks, dtype, mixed):
    """A prompt's rows, in tiles of every height, have the bits that they have in short batches; some of them in 64 bits too."""
    print(f"lora prompt tiles K={K} ranks={ranks} {dtype} mixed={mixed}", flush=True)
    gen = torch.Generator().manual_seed(K)
    T, outs = 1301, [32, 144, 16]
    store, a, b, scales = _store(K, outs, ranks, dtype, gen, dev, skip={(1, 1)})
    x = torch.randn((T, K), generator=gen).to(dtype).to(dev)
    y = torch.randn((T, sum(outs)), generator=gen).to(dtype).to(dev)
    rows = _rows(T, len(ranks), gen, mixed).to(dev)
    got = store.apply(x, y, rows, out=torch.empty_like(y))
    short = torch.cat([store.apply(x[t:t + 100], y[t:t + 100].clone(), rows[t:t + 100]) for t in range(0, T, 100)])
    assert torch.equal(got.view(torch.int16), short.view(torch.int16))
    some = torch.randperm(T, generator=gen)[:24].to(dev)
    _check(got[some], x[some], y[some], rows[some], a, b, scales, outs, dtype)


def test_lora_beside_dense_in_a_graph(dev):
    """As it is used: a trellis layer, then its adapters in place, captured once and replayed while the rows' adapters change
    and a slot is loaded anew; every replay equals the eager calls."""
    gen = torch.Generator().manual_seed(15)
    mats = [WL.matrix(512, n, 4, "int6", gen, dev) for n in (512, 128, 128)]
    layer, outs, K, T = Dn.Dense(mats), [512, 128, 128], 512, 7
    store, a, b, scales = _store(K, outs, [16, 8, 30], torch.bfloat16, gen, dev)
    x = torch.randn((T, K), generator=gen).to(torch.bfloat16).to(dev)
    rows, y = torch.zeros((T,), dtype=torch.int32, device=dev), torch.empty((T, 768), dtype=torch.bfloat16, device=dev)

    def step():
        layer.forward(x, out=y)
        store.apply(x, y, rows)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(4):
        ids = _rows(T, 3, gen)
        rows.copy_(ids)
        if k == 2:
            a[1] = [(torch.randn((12, K), generator=gen) / 16).to(torch.bfloat16) for _ in outs]
            b[1] = [torch.randn((n, 12), generator=gen).to(torch.bfloat16) for n in outs]
            store.load(1, a[1], b[1], scale=scales[1])
        g.replay()
        torch.cuda.synchronize()
        base = layer.forward(x)
        _check(y, x, base, ids, a, b, scales, outs, torch.bfloat16)
        eager = store.apply(x, base.clone(), rows)
        assert torch.equal(eager.view(torch.int16), y.view(torch.int16)), k


def test_lora_two_streams(dev):
    """Calls of two streams at once do not meet: each call has scratch of its own."""
    gen = torch.Generator().manual_seed(21)
    K, outs, T = 2048, [512], 64
    store, *_ = _store(K, outs, [64, 16], torch.bfloat16, gen, dev)
    xs = [torch.randn((T, K), generator=gen).to(torch.bfloat16).to(dev) for _ in range(2)]
    y = torch.randn((T, 512), generator=gen).to(torch.bfloat16).to(dev)
    rows = _rows(T, 2, gen).to(dev)
    want = [store.apply(x, y, rows, out=torch.empty_like(y)) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(20):
        for s, x, g in zip(streams, xs, got):
            with torch.cuda.stream(s):
                g.append(store.apply(x, y, rows, out=torch.empty_like(y)))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w.view(torch.int16), o.view(torch.int16)) for o in g)


def test_lora_loaded_from_views(dev):
    """Adapters given as transposed views, in another dtype and on the CPU or the device, in tiles that need no padding."""
    gen = torch.Generator().manual_seed(33)
    store = Adapters(64, [128], slots=2, max_rank=16, device=dev)
    a, b = torch.randn((64, 16), generator=gen), torch.randn((16, 128), generator=gen)
    store.load(0, [a.t()], [b.t()])
    store.load(1, [a.to(dev).t().contiguous().to(torch.bfloat16)], [b.to(dev).t()])
    assert torch.equal(store.a[0], store.a[1]) and torch.equal(store.b[0], store.b[1]) and store.b.any()


def test_lora_empty_and_refusals(dev, ext):
    gen = torch.Generator().manual_seed(30)
    store, *_ = _store(64, [32], [8], torch.bfloat16, gen, dev)
    x, y = torch.zeros((4, 64), dtype=torch.bfloat16, device=dev), torch.zeros((4, 32), dtype=torch.bfloat16, device=dev)
    rows = torch.zeros((4,), dtype=torch.int32, device=dev)
    assert store.apply(x[:0], y[:0], rows[:0]).shape == (0, 32)
    for args in ((x.half(), y, rows), (x, y.half(), rows), (x, y, rows.long()), (x, y, rows[:3]), (x[:, :32], y, rows),
                 (x, y[:, :16], rows), (x[:3], y, rows), (x.cpu(), y, rows), (x, y, rows.cpu()),
                 (x, torch.zeros((4, 34), dtype=torch.bfloat16, device=dev)[:, 2:], rows),
                 (x, torch.zeros((32, 4), dtype=torch.bfloat16, device=dev).t(), rows)):
        with pytest.raises(RuntimeError):
            store.apply(*args)
    with pytest.raises(RuntimeError):
        ext.lora(x, y, y, rows, store.a, store.b[:, :0], store.ranks, store.scales, [32])
    with pytest.raises(RuntimeError):
        ext.lora(x, y, y, rows, store.a, store.b, store.ranks, store.scales, [16, 16])
