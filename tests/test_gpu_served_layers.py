"""GPU checks of a synthetic decoder whose layers differ in what stands beside and behind them (vllm_espalier/step.py): adapters at
qkv or at o alone, in a later layer alone, a norm behind one block alone. Every such decoder has the logits of one that has all
of it, empty where the first has nothing, bit for bit; and rows alone (whose norms may run inside the launches) have the bits that
they have in a window (whose norms run apart) and, adapters in place, not the plain decoder's."""
import pytest
import torch

from vllm_espalier import step as S
from vllm_espalier.adapters import Adapters

pytestmark = pytest.mark.gpu
VOCAB, SLOTS, RANK = 5120, 2, 12
IDS, ROWS = [5, 4095, 17, 300, 2, 800], [0, 1, -1, 1, 0, 0]


def _fill(store, seed):
    gen = torch.Generator().manual_seed(seed)
    K = store.in_features
    for slot in range(SLOTS):
        store.load(slot, [(torch.randn((RANK, K), generator=gen) * K ** -0.5).to(torch.bfloat16) for _ in store.out_features],
                   [(torch.randn((n, RANK), generator=gen) * RANK ** -0.5).to(torch.bfloat16) for n in store.out_features], 0.5)


def _decoder(dev):
    return S.SyntheticDecoder(n_layers=2, seed=9, device=dev, E=16, vocab=VOCAB)


def _run(dec, rows=slice(None), prompt=False):
    ids, slots = IDS[rows], ROWS[rows]
    T = len(ids)
    b = dec.prefill_buffers(T) if prompt else dec.buffers(T)
    b.ids_in.copy_(torch.tensor(ids, dtype=torch.int32))
    b.rows.copy_(torch.tensor(slots, dtype=torch.int32))
    dec.prefill(T, head_rows=T) if prompt else dec.forward(T)
    torch.cuda.synchronize()
    return b.logits.clone().view(torch.int16)


@pytest.mark.parametrize("layer,where", [(0, "qkv"), (0, "o"), (1, "qkv"), (1, "o"), (1, "both")])
def test_adapters_at_one_place(dev, layer, where):
    print(f"adapters at layer {layer}, {where}", flush=True)
    dec, full = _decoder(dev), _decoder(dev)
    plain = _run(dec)
    full.use_adapters(SLOTS, RANK)
    stores = {"qkv": (Adapters(S.D_MODEL, [S.Q_OUT, S.KV_OUT, S.KV_OUT], SLOTS, RANK, device=dev), full.layers[layer].qkv_adapters),
              "o": (Adapters(S.Q_OUT, [S.D_MODEL], SLOTS, RANK, device=dev), full.layers[layer].o_adapters)}
    for i, name in enumerate(stores):
        if where in (name, "both"):
            for store in stores[name]:
                _fill(store, i)
            setattr(dec.layers[layer], name + "_adapters", stores[name][0])
    whole = _run(dec)
    assert torch.equal(whole, _run(full)) and not torch.equal(whole, plain)
    assert torch.equal(whole[2], plain[2])                   # a row of no adapter
    assert torch.equal(_run(dec, prompt=True), _run(full, prompt=True))
    for r in range(len(IDS)):                                # decode of one row and of three
        assert torch.equal(_run(dec, slice(r, r + 1)), whole[r:r + 1]), r
    assert torch.equal(_run(dec, slice(1, 4)), whole[1:4])
    assert not dec.fused_norms(1)


@pytest.mark.parametrize("layer,name", [(0, "post_o"), (1, "post_in"), (1, "post_o")])
def test_one_norm_behind_a_block(dev, layer, name):
    print(f"{name} at layer {layer}", flush=True)
    dec = _decoder(dev)
    plain = _run(dec)
    gen = torch.Generator(device=dev).manual_seed(4)
    setattr(dec.layers[layer], name, S._norm_weight(gen, dev, S.D_MODEL))
    whole = _run(dec)
    assert not torch.equal(whole, plain)
    for r in range(len(IDS)):
        assert torch.equal(_run(dec, slice(r, r + 1)), whole[r:r + 1]), r
    assert torch.equal(_run(dec, slice(1, 4)), whole[1:4])
    assert not dec.fused_norms(1)


def test_plain_layers_stay_fused(dev, monkeypatch):
    """Beside a layer with adapters the others keep their launches, and everything has the bits of the launches apart."""
    dec = _decoder(dev)
    dec.layers[1].o_adapters = Adapters(S.Q_OUT, [S.D_MODEL], SLOTS, RANK, device=dev)
    _fill(dec.layers[1].o_adapters, 1)
    assert dec._fused(dec.layers[0], 1) and not dec._fused(dec.layers[1], 1)
    got = _run(dec, slice(0, 1))
    monkeypatch.setattr(S, "FUSE_NORMS", False)
    monkeypatch.setattr(S, "MULTI_ATTN", False)
    assert torch.equal(_run(dec, slice(0, 1)), got)


def test_algorithmic_bytes_count_every_norm(dev):
    """The weights of the norms behind the blocks: two a layer, of which the last MoE's runs before the head."""
    picks = [torch.empty((0,), dtype=torch.int32)] * 2
    plain, posts = _decoder(dev), S.SyntheticDecoder(n_layers=2, seed=9, device=dev, E=16, vocab=VOCAB, post_norms=True)
    assert posts.algorithmic_bytes(picks, 3) - plain.algorithmic_bytes(picks, 3) == 4 * S.D_MODEL * 2
    assert posts.algorithmic_bytes(picks, 3, head=False) - plain.algorithmic_bytes(picks, 3, head=False) == 3 * S.D_MODEL * 2
