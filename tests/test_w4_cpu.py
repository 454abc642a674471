"""Modules with 4-bit weights without a GPU: what replacing a model's layers and
moving them between types leaves."""

import pytest
import torch
import torch.nn as nn

from conftest import load_pkg

w4 = load_pkg().w4


def host_weight(out, d_in, group=64):
    n, k = -(-out // 16), -(-d_in // 128)
    g = torch.Generator().manual_seed(out)
    packed = torch.randint(0, 256, (n, k, 4, 16, 16), generator=g).to(torch.uint8)
    scales = torch.rand(n, k, 16, 128 // group, generator=g).to(torch.bfloat16)
    return w4.W4Weight(packed, scales, out, d_in, group)


@pytest.fixture
def quantize_on_the_host(monkeypatch):
    """Codes and scales that have nothing to do with the weight; nothing computes with them."""
    monkeypatch.setattr(w4, "quantize", lambda weight, group: host_weight(*weight.shape, group))


def test_every_name_of_a_layer_is_replaced(quantize_on_the_host):
    a, b = nn.Linear(8, 8, bias=False), nn.Linear(8, 4, bias=False)
    model = nn.Sequential(a, b, a)
    model.inner = nn.Module()
    model.inner.first, model.inner.second = b, b
    w4.quantize_model(model, 64)
    assert type(model[0]) is type(model[1]) is w4.W4Linear
    assert model[2] is model[0] and model.inner.first is model.inner.second is model[1]
    assert not any(isinstance(m, nn.Linear) for m in model.modules())


def test_a_layer_that_cannot_be_quantised_leaves_the_model_whole(monkeypatch):
    def quantize(weight, group):
        if weight.dtype != torch.float32:
            raise TypeError("expected float32 or bfloat16")
        return host_weight(*weight.shape, group)
    monkeypatch.setattr(w4, "quantize", quantize)
    model = nn.Sequential(nn.Linear(8, 8, bias=False), nn.Linear(8, 8, bias=False).half())
    kept = list(model)
    with pytest.raises(TypeError):
        w4.quantize_model(model, 64)
    assert list(model) == kept


@pytest.mark.parametrize("cast", [lambda m: m.float(), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.bfloat16(), lambda m: m.to(torch.float32), lambda m: m.type(torch.float32),
                                  lambda m: m.half().float(), lambda m: m.to("cpu")])
def test_casting_a_model_leaves_the_format(cast):
    """Scales of up to the largest bf16 number, which fp16 does not hold."""
    w = host_weight(20, 130, 32)
    w.scales[0, 0, 0, 0], w.scales[0, 0, 1, 0] = 3e38, 1e-38
    model = nn.Sequential(nn.Linear(4, 130), w4.W4Linear(w))
    packed, scales = w.packed.clone(), w.scales.clone()
    cast(model)
    got = model[1].weight                                            # W4Weight checks the types
    assert torch.equal(got.packed, packed) and torch.equal(got.scales, scales)
    assert set(dict(model[1].named_buffers())) == {"packed", "scales"}
    assert got.packed.data_ptr() == model[1].packed.data_ptr()


def test_a_moved_model_keeps_the_format():
    model = nn.Sequential(w4.W4Linear(host_weight(20, 130, 32)))
    model.to("meta", torch.float16)
    assert model[0].scales.device.type == "meta" and model[0].scales.dtype == torch.bfloat16
    model.to_empty(device="cpu")
    assert model[0].weight.scales.shape == (2, 2, 16, 4)
