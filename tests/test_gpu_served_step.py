"""GPU checks of the adapters, the norms around a block and the verification together, as a served step runs them: a synthetic
decoder whose blocks have norms behind them and whose requests have adapters verifies their drafts (vllm_espalier/step.py), and
a vLLM-style linear layer with adapters attached (vllm_espalier/linear.py).

Bars: rows without adapters give the plain decoder's bits; rows alone give the bits of the same rows in a window, in a graph
those of the eager call; tokens follow the rule in 64 bits from the logits, where it decides by more than 1e-5.
"""
import pytest
import torch

from test_gpu_verify import _check as check_verify
from vllm_espalier import linear as LN
from vllm_espalier import step as S
from vllm_espalier import workloads as WL

pytestmark = pytest.mark.gpu
VOCAB, SLOTS, RANKS = 5120, 3, [16, 5, 24]


def _load(dec, seed):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *shape, by: (torch.randn(shape, generator=gen) * by).to(torch.bfloat16)  # noqa: E731
    for L in dec.layers:
        for store in (L.qkv_adapters, L.o_adapters):
            K = store.in_features
            for slot, r in enumerate(RANKS):
                store.load(slot, [rnd(r, K, by=K ** -0.5) for _ in store.out_features],
                           [rnd(n, r, by=r ** -0.5) for n in store.out_features], scale=0.5)


@pytest.fixture(scope="module")
def decoder(dev):
    dec = S.SyntheticDecoder(n_layers=2, seed=9, device=dev, E=16, vocab=VOCAB, post_norms=True)
    dec.use_adapters(SLOTS, max(RANKS))
    _load(dec, 1)
    return dec


def _run(dec, ids, rows):
    b = dec.buffers(len(ids))
    b.ids_in.copy_(torch.tensor(ids, dtype=torch.int32))
    b.rows.copy_(torch.tensor(rows, dtype=torch.int32))
    dec.forward(len(ids))
    torch.cuda.synchronize()
    return b


def test_rows_without_adapters_are_the_plain_step(dev):
    """Adapters that no row names, and no norms behind the blocks: the plain decoder's logits bit for bit, decode and prefill."""
    plain = S.SyntheticDecoder(n_layers=2, seed=9, device=dev, E=16, vocab=VOCAB)
    ids = [5, 4095, 17]
    want = _run(plain, ids, [-1] * 3).logits.clone()
    pb = plain.prefill_buffers(40)
    pb.ids_in.copy_(torch.arange(40, dtype=torch.int32) * 7)
    prompt = plain.prefill(40, head_rows=40).logits.clone()
    plain.use_adapters(SLOTS, max(RANKS))
    _load(plain, 1)
    assert torch.equal(_run(plain, ids, [-1] * 3).logits.view(torch.int16), want.view(torch.int16))
    pb.rows.fill_(-1)
    assert torch.equal(plain.prefill(40, head_rows=40).logits.view(torch.int16), prompt.view(torch.int16))
    assert not torch.equal(_run(plain, ids, [0, 1, 2]).logits, want)


def test_rows_alone_equal_window(decoder):
    ids, rows = [5, 4095, 17, 300, 2, 2, 800], [0, -1, 2, 1, 1, 0, 2]
    b = _run(decoder, ids, rows)
    logits, h = b.logits.clone(), b.h.clone()
    assert torch.isfinite(logits.float()).all()
    for r in range(len(ids)):
        one = _run(decoder, ids[r:r + 1], rows[r:r + 1])
        assert torch.equal(one.logits.view(torch.int16), logits[r:r + 1].view(torch.int16)), r
        assert torch.equal(one.h.view(torch.int16), h[r:r + 1].view(torch.int16)), r


def test_prefill_rows_alone_equal_prompt(decoder):
    T = 70
    b = decoder.prefill_buffers(T)
    ids = [(11 + 977 * i) % VOCAB for i in range(T)]
    rows = [0] * 20 + [2] * 25 + [-1] * 3 + [1] * 22
    b.ids_in.copy_(torch.tensor(ids, dtype=torch.int32))
    b.rows.copy_(torch.tensor(rows, dtype=torch.int32))
    logits = decoder.prefill(T, head_rows=T).logits.clone()
    assert torch.isfinite(logits.float()).all()
    one = decoder.prefill_buffers(1)
    for r in (0, 19, 20, 46, 69):
        one.ids_in.fill_(ids[r])
        one.rows.fill_(rows[r])
        assert torch.equal(decoder.prefill(1).logits.view(torch.int16), logits[r:r + 1].view(torch.int16)), r


def _requests(dev, gen, logits_rows):
    """Three requests over 9 rows: 3 drafts, 1 draft, 2 drafts; the second greedy."""
    n = torch.tensor([3, 1, 2], dtype=torch.int32)
    first = torch.tensor([0, 4, 6], dtype=torch.int32)
    assert logits_rows == 9
    return {"first": first.to(dev), "n": n.to(dev),
            "drafts": torch.randint(0, VOCAB, (3, 3), generator=gen, dtype=torch.int32).to(dev),
            "uniform": torch.rand((3, 3), generator=gen).to(dev),
            "race": torch.empty((3, VOCAB)).exponential_(generator=gen).to(dev),
            "temp": torch.tensor([0.9, 0.0, 1.2]).to(dev),
            "probs": torch.softmax(torch.randn((3, 3, VOCAB), generator=gen) * 3, -1).to(dev)}


def test_verify_step_eager_and_graph(dev, decoder):
    """A pass over last tokens and drafts, then their verification: by the rule, and replayed with other tokens, rows and random
    numbers the eager results."""
    gen = torch.Generator().manual_seed(3)
    q = _requests(dev, gen, 9)
    b = decoder.buffers(9)

    def step():
        decoder.forward(9)
        return decoder.verify(b, q["first"], q["n"], q["drafts"], q["uniform"], q["race"], q["temp"], draft_probs=q["probs"])

    def new_inputs(k):
        b.ids_in.copy_(torch.randint(0, VOCAB, (9,), generator=gen, dtype=torch.int32))
        b.rows.copy_(torch.tensor([0] * 4 + [-1] * 2 + [k % SLOTS] * 3, dtype=torch.int32))
        q["uniform"].copy_(torch.rand((3, 3), generator=gen))
        q["race"].copy_(torch.empty((3, VOCAB)).exponential_(generator=gen))
        # drafts that the target may accept: its own likeliest tokens at these rows, for the greedy request among them
        decoder.forward(9)
        top = b.logits.float().argmax(-1).to(torch.int32)
        q["drafts"][0, 0], q["drafts"][1, 0], q["drafts"][2, :2] = top[0], top[4], top[6:8]

    new_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    accepted = 0
    for k in range(4):
        new_inputs(k)
        g.replay()
        torch.cuda.synchronize()
        logits, got = b.logits.clone(), [t.clone() for t in out]
        eager = step()
        assert torch.equal(b.logits.view(torch.int16), logits.view(torch.int16)), k
        assert all(torch.equal(x, y) for x, y in zip(got, eager)), k
        check_verify({"logits": logits.cpu(), **{n: t.cpu() for n, t in q.items()}}, [t.cpu() for t in got], few=0.4)
        accepted += int((got[1] - 1).sum())
    assert accepted >= 4                                     # the greedy request's draft every time


@pytest.mark.parametrize("fused", [True, False])
def test_linear_layer_with_adapters(dev, fused):
    gen = torch.Generator().manual_seed(8)
    mats = [WL.matrix(256, n, 4, "int6", gen, dev) for n in (256, 128)]
    layer = LN.TrellisLinear(mats, 384 + 16, fused)
    x = torch.randn((2, 5, 256), generator=gen).to(torch.bfloat16).to(dev)
    rows = torch.tensor([[0, 1, -1, 0, 1], [1, 1, 0, -1, 5]], dtype=torch.int32, device=dev)
    base = layer(x)
    with pytest.raises(RuntimeError):
        layer(x, rows)
    store = layer.attach_adapters(2, 12)
    a = [[(torch.randn((r, 256), generator=gen) / 16).to(torch.bfloat16) for _ in mats] for r in (12, 3)]
    b = [[torch.randn((n, r), generator=gen).to(torch.bfloat16) for n in (256, 128)] for r in (12, 3)]
    for i in range(2):
        store.load(i, a[i], b[i], scale=0.25)
    assert torch.equal(layer(x).view(torch.int16), base.view(torch.int16))
    y = LN.EspLinearMethod("q").apply(type("Layer", (), {"espalier": layer})(), x, adapter_rows=rows)
    assert y.shape == base.shape and torch.equal(y[..., 384:], base[..., 384:])
    want = store.apply(x.view(10, 256), base.view(10, 400).clone(), rows.view(-1))
    assert torch.equal(y.view(10, 400).view(torch.int16), want.view(torch.int16))
    assert torch.equal(y[0, 2].view(torch.int16), base[0, 2].view(torch.int16)) and not torch.equal(y[0, 0], base[0, 0])
