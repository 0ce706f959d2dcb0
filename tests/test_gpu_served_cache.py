"""GPU checks of the paged cache, the attention over it and the token log-probabilities together, as a served step runs them: a
synthetic decoder prefills requests into its caches, decodes them with drafts and without, eagerly and in a graph, and scores tokens
(vllm_espalier/step.py). What the cache holds and what o reads are compared with plain forms in 64 bits (paged.py)."""
import pytest
import torch

import paged
from test_gpu_attention import compare
from test_gpu_logprobs import check as check_logprobs
from vllm_espalier import step as S

pytestmark = pytest.mark.gpu
VOCAB, PAGE, PAGES = 5120, 32, 40


def _decoder(dev, layers=2, **more):
    dec = S.SyntheticDecoder(n_layers=layers, seed=9, device=dev, E=16, vocab=VOCAB)
    dec.use_cache(PAGES, PAGE, **more)
    return dec


@pytest.fixture(scope="module")
def decoder(dev):
    return _decoder(dev, split=128)


TABLES = [[7, 3, 30, 12], [1, 2], [39, 0, 5], [20, 21, 22, 23]]


def _run(dec, ids, lengths, n_new, tables=TABLES, max_new=4):
    """A decode pass over requests' new tokens."""
    T = len(ids)
    b = dec.buffers(T)
    s = dec.sequences(b, requests=len(lengths), max_new=max_new, pages=5)
    s.place(tables[:len(lengths)], lengths, n_new)
    b.ids_in.copy_(torch.tensor(ids, dtype=torch.int32))
    dec.forward(T)
    torch.cuda.synchronize()
    return b


def _prefill(dec, prompts, head_rows=1):
    T = sum(prompts)
    b = dec.prefill_buffers(T)
    dec.sequences(b, requests=len(prompts), max_new=max(prompts), pages=5).place(TABLES[:len(prompts)], prompts, prompts)
    b.ids_in.copy_((torch.arange(T) * 977 + 11) % VOCAB)
    dec.prefill(T, head_rows=head_rows)
    torch.cuda.synchronize()
    return b


def _check_last_layer(dec, b, lengths, n_new):
    """The last layer's cache against its k and v, and what o read against its turned q."""
    L, s = dec.layers[-1], b.sequences
    q, k, v = (t.reshape(b.T, -1, S.HEAD_DIM) for t in b.qkv.split([S.Q_OUT, S.KV_OUT, S.KV_OUT], dim=1))
    kv = paged.cache_values(L.cache)
    slots = s.slots.cpu()
    here = slots >= 0
    want = paged.turned(k, L.k_norm, s.positions, dec.rotary, S.EPS)[here]
    compare(kv[0][slots[here] // PAGE, slots[here] % PAGE], want, paged.turned_bound(None, None, want, torch.bfloat16))
    assert torch.equal(kv[1][slots[here] // PAGE, slots[here] % PAGE], v.double().cpu()[here])
    first = [sum(n_new[:i]) for i in range(len(n_new))]
    want, bound, rows = paged.attention(q, kv, s.tables, lengths, first, n_new, S.HEAD_DIM ** -0.5)
    compare(b.attn.view(b.T, -1, S.HEAD_DIM), want, bound, rows)


def test_prefill_then_decode(decoder):
    prompts = [90, 33, 1]
    b = _prefill(decoder, prompts, head_rows=124)
    assert torch.isfinite(b.logits.float()).all()
    _check_last_layer(decoder, b, prompts, prompts)
    lengths = list(prompts)
    for n_new in ([1, 1, 1], [4, 1, 2], [3, 2, 4]):
        lengths = [v + n for v, n in zip(lengths, n_new)]
        b = _run(decoder, [(5 + 31 * i) % VOCAB for i in range(sum(n_new))], lengths, n_new)
        assert torch.isfinite(b.logits.float()).all()
        _check_last_layer(decoder, b, lengths, n_new)
        tokens = torch.arange(b.T, dtype=torch.int32, device=b.logits.device) * 501 % VOCAB
        got = decoder.score(b, tokens, top=4)
        want = check_logprobs(b.logits, tokens, 4)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.equal(got[3][:, 0], b.ids_out)           # the likeliest is what the decoder takes


def test_requests_alone_equal_batch(decoder):
    """With a split of its own a request's rows have the bits that they have alone, prompts and drafts both."""
    prompts = [90, 33, 60]
    _prefill(decoder, prompts)
    lengths, n_new = [94, 34, 63], [4, 1, 3]
    ids = [(17 + 131 * i) % VOCAB for i in range(8)]
    logits = _run(decoder, ids, lengths, n_new).logits.clone()
    at = 0
    for r, n in enumerate(n_new):
        one = _run(decoder, ids[at:at + n], lengths[r:r + 1], [n], tables=TABLES[r:])
        assert torch.equal(one.logits.view(torch.int16), logits[at:at + n].view(torch.int16)), r
        at += n


def test_a_drafted_token_equals_a_decoded_one(decoder):
    """Tokens one at a time give the bits of the same tokens as drafts: their keys and values are the same, whoever stands beside."""
    _prefill(decoder, [90])
    ids = [5, 4095, 17, 300]
    together = _run(decoder, ids, [94], [4]).logits.clone()
    for i, t in enumerate(ids):
        one = _run(decoder, [t], [91 + i], [1]).logits
        assert torch.equal(one.view(torch.int16), together[i:i + 1].view(torch.int16)), i


@pytest.mark.parametrize("eight", [False, True])
def test_graph_of_a_step(dev, eight):
    """A captured decode step, replayed over growing requests with padding among the rows, between eager passes; the score of its
    tokens in the graph too."""
    dec = _decoder(dev, dtype=torch.float8_e4m3fn, scale=0.03) if eight else _decoder(dev)
    _prefill(dec, [90, 33, 1])
    b = dec.buffers(4)
    s = dec.sequences(b, max_new=1, pages=5)
    tokens = torch.zeros((4,), dtype=torch.int32, device=dev)

    def step():
        dec.forward(4)
        return dec.score(b, tokens, top=3)

    def new(k):
        n = 3 if k % 2 else 2
        s.place(TABLES[:n], [91 + k, 34 + k, 2 + k][:n])
        b.ids_in.copy_(torch.tensor([k, 2 * k, 3 * k, 0], dtype=torch.int32))
        tokens.copy_(torch.tensor([k, 100 * k, VOCAB - 1 - k, -1], dtype=torch.int32))

    new(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(1, 6):
        new(k)
        g.replay()
        torch.cuda.synchronize()
        n = int((s.n_new > 0).sum())
        logits, got = b.logits[:n].clone(), [t[:n].clone() for t in out]
        assert torch.isfinite(logits.float()).all()
        eager = step()
        assert torch.equal(b.logits[:n].view(torch.int16), logits.view(torch.int16))
        assert all(torch.equal(x, y[:n]) for x, y in zip(got, eager))


def test_a_decoder_without_a_cache_is_as_before(dev):
    plain = S.SyntheticDecoder(n_layers=2, seed=9, device=dev, E=16, vocab=VOCAB)
    b = plain.buffers(3)
    b.ids_in.copy_(torch.tensor([5, 4095, 17], dtype=torch.int32))
    want = plain.forward(3).logits.clone()
    plain.use_cache(PAGES, PAGE)
    with pytest.raises(RuntimeError, match="sequences"):
        plain.forward(3)
    for L in plain.layers:
        L.cache = None
    assert torch.equal(plain.forward(3).logits, want)
