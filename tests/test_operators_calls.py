"""Calls of the adapters, the verification and the norms around a block that have to be refused, or must leave nothing behind, on
the CPU: the package's own checks in front of the extension, and the C ABI's before any HIP call."""
import pytest
import torch

from vllm_espalier import linear as LN
from vllm_espalier.adapters import Adapters


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
