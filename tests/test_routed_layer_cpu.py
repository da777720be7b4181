"""What MoELayer.forward_routed refuses and what it hands on, with stand-ins for the operators: no device is needed."""
import pytest
import torch

from ascend_kernel_b200 import moe_layer as ml


def _layer(fmt):
    layer = object.__new__(ml.MoELayer)
    layer.world, layer.px, layer.weight_format, layer.n_experts, layer.hidden = 1, None, fmt, 4, 8
    return layer


def _stand_ins(monkeypatch, calls):
    def sort(idx, n):
        flat = idx.reshape(-1).long()
        order = flat.sort(stable=True).indices
        slot = torch.empty_like(flat)
        slot[order] = torch.arange(flat.numel())
        return torch.bincount(flat, minlength=n), (order // idx.shape[1]).to(torch.int32), slot.view_as(idx).to(torch.int32)

    rows = lambda x, token_of, *_: (torch.zeros(token_of.numel(), x.shape[1]), None)  # noqa: E731
    monkeypatch.setattr(ml.ops, "moe_sort", sort)
    monkeypatch.setattr(ml.ops, "fp8_quantize_rows", rows)
    monkeypatch.setattr(ml.ops, "mxfp4_quantize_rows", rows)
    monkeypatch.setattr(ml.ops, "moe_dispatch", lambda x, token_of, slot: rows(x, token_of)[0])
    monkeypatch.setattr(ml.ops, "moe_combine", lambda y, weight, token_of, slot: y.new_zeros(slot.shape[0], y.shape[1]))

    def experts(self, send, counts, record, **kw):
        calls.append((send, counts, kw))
        return send

    monkeypatch.setattr(ml.MoELayer, "_experts", experts)


@pytest.mark.parametrize("fmt", ["int8", "fp4", "fp8", "mxfp4"])
@pytest.mark.parametrize("tokens", [2, 4])
def test_a_choice_for_other_tokens_is_refused(monkeypatch, fmt, tokens):
    calls = []
    _stand_ins(monkeypatch, calls)
    layer, x = _layer(fmt), torch.zeros(3, 8, dtype=torch.bfloat16)
    good = torch.zeros(3, 2, dtype=torch.int32)
    assert layer.forward_routed(x, good, torch.ones(3, 2)).shape == (3, 8) and len(calls) == 1
    with pytest.raises(RuntimeError, match="tokens"):
        layer.forward_routed(x, torch.zeros(tokens, 2, dtype=torch.int32), torch.ones(tokens, 2))
    with pytest.raises(RuntimeError, match="tokens"):
        layer.forward_routed(x, good, torch.ones(tokens, 2))
    assert len(calls) == 1


def test_rows_an_expert_has_at_most(monkeypatch):
    """A token may name an expert more than once, so that an expert has more rows than there are tokens: no such bound is handed on."""
    calls = []
    _stand_ins(monkeypatch, calls)
    layer = _layer("int8")
    layer.forward_routed(torch.zeros(5, 8, dtype=torch.bfloat16), torch.full((5, 3), 2, dtype=torch.int32), torch.ones(5, 3))
    _, counts, kw = calls[0]
    assert int(counts.max()) == 15
    assert kw.get("max_rows") is None or kw["max_rows"] >= 15
