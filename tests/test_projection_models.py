"""Models with 8-bit projections and adapters that a step could not run are refused when
they are made (CPU): a step that fails half way has bound blocks and written K and V."""
from types import SimpleNamespace

import pytest
import torch

from zealot_amd import dense
from zealot_amd.model import HipModelRunner, LayerAdapters, LayerWeights, LlamaAdapters, LlamaConfig, LlamaWeights

BF, F32 = torch.bfloat16, torch.float32


def _weights(cfg, dtype=BF):
    z = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    H, Hkv, D, hid, I = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.hidden_size, cfg.intermediate_size
    layer = LayerWeights(z(hid), z((H + 2 * Hkv) * D, hid), z(hid, H * D), z(hid), z(2 * I, hid), z(hid, I))
    return LlamaWeights(z(8, hid), [layer] * cfg.num_layers, z(hid), z(8, hid))


def _packed(n, k):
    size = -(-n // 64) * 4 * -(-k // 128) * 2048
    return dense.Fp8Weight(torch.zeros(size, dtype=torch.uint8), torch.ones(n), n, k)


def _cfg(hidden=64, inter=96, layers=2):
    return LlamaConfig(8, hidden, inter, layers, 2, 1, 64)


def _runner(cfg, w, ad=None):
    kv = SimpleNamespace(cache=SimpleNamespace(num_layers=cfg.num_layers, num_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim))
    return HipModelRunner(cfg, w, kv, ad)


@pytest.mark.parametrize("hidden,inter,what", [(64, 53248, "intermediate"), (64, 4112 - 8, "intermediate"), (72, 96, "hidden"), (33024, 96, "hidden")])
def test_sizes_that_have_no_8_bit_rows(hidden, inter, what):
    w = _weights(_cfg(hidden, inter, 1))
    with pytest.raises(ValueError, match=what):
        w.in_8_bits()
    # weights packed by hand
    cfg = _cfg(hidden, inter, 1)
    lw = w.layers[0]
    lw.qkv, lw.gate_up, lw.down = (_packed(*t.shape) for t in (lw.qkv, lw.gate_up, lw.down))
    with pytest.raises(ValueError, match=what):
        _runner(cfg, w)


def test_some_weights_in_8_bits():
    cfg = _cfg()
    w = _weights(cfg)
    assert not _runner(cfg, w).in_8_bits
    from dataclasses import replace
    one = replace(w.layers[0], **{k: _packed(*getattr(w.layers[0], k).shape) for k in ("qkv", "gate_up", "down")})
    assert _runner(cfg, replace(w, layers=[one, one])).in_8_bits
    for layers in ([one, w.layers[0]], [one, replace(one, down=w.layers[0].down)], [one, replace(one, qkv=w.layers[0].qkv)]):
        with pytest.raises(ValueError, match="every layer"):
            _runner(cfg, replace(w, layers=layers))


def _adapters(cfg, dtype=F32, count=3, rank=4):
    return LlamaAdapters.random(cfg, count, rank, dtype, device="cpu")


def test_adapters_that_fit():
    cfg = _cfg()
    for dtype in (F32, BF):
        _runner(cfg, _weights(cfg, dtype), _adapters(cfg, dtype))
    ad = _adapters(cfg)
    ad.scales = None
    ad.layers = [LayerAdapters(), LayerAdapters(o=ad.layers[0].o)]
    _runner(cfg, _weights(cfg, F32), ad)


@pytest.mark.parametrize("count,rank", [(2049, 1), (1, 257), (1, 171), (2, 0)])
def test_adapters_over_the_operators_limits(count, rank):
    """2048 adapters, 256 ranks of a part, 512 of all (q, k and v have three)."""
    cfg = _cfg(layers=1)
    w = _weights(cfg, F32)
    with pytest.raises(ValueError, match="dense.lora"):
        _runner(cfg, w, _adapters(cfg, F32, count, rank))


def test_adapters_of_another_model():
    cfg = _cfg()
    w = _weights(cfg, F32)
    with pytest.raises(TypeError):
        _runner(cfg, w, _adapters(cfg, BF))
    for other in (_cfg(hidden=128), _cfg(inter=128)):
        with pytest.raises(ValueError):
            _runner(cfg, w, _adapters(other))
    for name in ("qkv", "o", "gate_up", "down"):
        for i in (0, 1):
            ad = _adapters(cfg)
            pair = list(getattr(ad.layers[1], name))
            pair[i] = pair[i][:2]
            setattr(ad.layers[1], name, tuple(pair))
            with pytest.raises(ValueError, match=f"layer 1: {'ab'[i]} of {name}"):
                _runner(cfg, w, ad)
    ad = _adapters(cfg)
    a, b = ad.layers[0].o
    ad.layers[0].o = (a, b.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="contiguous"):
        _runner(cfg, w, ad)
    ad = _adapters(cfg)
    ad.scales = ad.scales[:2]
    with pytest.raises(ValueError, match="scales"):
        _runner(cfg, w, ad)
    ad.scales = torch.ones(3, dtype=torch.float64)
    with pytest.raises(TypeError, match="scales"):
        _runner(cfg, w, ad)


def test_adapters_are_named_by_whole_numbers():
    """A step's rows take the adapter that its request names, and nothing near it."""
    import numpy as np
    cfg = _cfg()
    runner = _runner(cfg, _weights(cfg, F32), _adapters(cfg))
    out = SimpleNamespace(batch=[SimpleNamespace(request_id="a", num_tokens=2), SimpleNamespace(request_id="b", num_tokens=1)])
    assert runner._adapter_rows(out, {"a": 1}) == [1, 1, -1]
    assert runner._adapter_rows(out, {"a": np.int64(2), "b": torch.tensor(0)}) == [2, 2, 0]
    assert runner._adapter_rows(out, {"b": None, "c": 7}) is None
    for bad in (0.5, 1.0, "1", np.float32(1)):
        with pytest.raises(TypeError):
            runner._adapter_rows(out, {"a": bad})
    for bad in (-1, 3):
        with pytest.raises(ValueError):
            runner._adapter_rows(out, {"a": bad})
