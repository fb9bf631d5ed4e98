"""Host-side behaviour of the models and layers around the RACE layer (runs without a GPU)."""
import subprocess
import sys
import weakref

import pytest
import torch

from conftest import ROOT


def _int8_linear():
    """An Int8Linear of given rows (its constructor quantises on the GPU)."""
    from race_attention_b200 import Int8Linear
    layer = Int8Linear.__new__(Int8Linear)
    torch.nn.Module.__init__(layer)
    layer.out_features, layer.in_features, layer.dtype = 3, 16, torch.bfloat16
    layer.register_buffer("q", torch.arange(48, dtype=torch.int8).view(3, 16))
    layer.register_buffer("scale", torch.tensor([0.1, 0.3, 1 / 3]))
    layer.register_buffer("bias", torch.tensor([0.7, -0.1, 1 / 7]))
    return layer


def test_int8_layer_keeps_its_scales_when_converted():
    layer = _int8_linear()
    want = {k: v.clone() for k, v in layer.state_dict().items()}
    for kind in (torch.bfloat16, torch.float16, torch.float64, torch.float32):
        moved = layer.to(kind)
        assert moved is layer
        assert all(torch.equal(want[k], v) and want[k].dtype == v.dtype for k, v in layer.state_dict().items())


def test_int8_layer_leaves_the_meta_device():
    layer = _int8_linear()
    held = {k: v.clone() for k, v in layer.state_dict().items()}
    layer.to(torch.bfloat16).to("meta")
    assert all(v.device.type == "meta" for v in layer.state_dict().values())
    layer.to_empty(device="cpu")
    layer.load_state_dict(held)
    assert all(torch.equal(held[k], v) and held[k].dtype == v.dtype for k, v in layer.state_dict().items())
    assert layer.q.device.type == layer.scale.device.type == layer.bias.device.type == "cpu"


def test_package_imports_where_torch_has_no_cuda():
    """What needs no GPU (planes, the host's part of the shard exchange) works with a torch built without CUDA."""
    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_get")]:
    delattr(torch._C, name)
import race_attention_b200 as rb
planes, _ = rb.build_planes_protos(64, 4, 16, 1, device="cpu", seed=0)
assert planes.isfinite().all()
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


def _hybrid():
    from race_attention_b200.hybrid import HybridConfig, HybridLlama
    torch.manual_seed(0)
    return HybridLlama(HybridConfig(vocab_size=50, n_layer=2, hidden=64, n_head=2, n_kv_head=1, mlp_hidden=64))


def test_prefill_lets_go_of_each_slice(monkeypatch):
    """No hidden state of one slice of the batch is held while the next one is worked on."""
    model, seen = _hybrid(), []

    def hidden(x, cos, sin, t_max, b0, batch):
        assert not any(r() is not None for r in seen), "an earlier slice is still held"
        seen.append(weakref.ref(x))
        return lambda at: x[:, at]

    monkeypatch.setattr(model, "_prefill_hidden", hidden)
    assert model.prefill(torch.zeros(6, 5, dtype=torch.int64), t_max=8, micro_batch=2).shape == (6,)
    assert len(seen) == 3


def test_scoring_that_fails_leaves_the_decode_state(monkeypatch):
    """A forward that stops half-way (out of memory, say) leaves every layer's state and cache as they were."""
    model = _hybrid()
    for layer in model.layers:
        layer.state, layer.cache, layer.attn_ws, layer.n_splits = object(), (object(), object()), object(), 7
    held = [(a.state, a.cache, a.attn_ws, a.n_splits) for a in model.layers]

    def first(x, cos, sin, t_max, b0, batch):
        layer = model.layers[0]
        layer.state, layer.cache, layer.attn_ws, layer.n_splits = None, None, None, 1
        return x

    def second(x, *a):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(model.layers[0], "prefill", first)
    monkeypatch.setattr(model.layers[1], "prefill", second)
    for call in (model.score, model.logits_full):
        with pytest.raises(RuntimeError, match="out of memory"):
            call(torch.zeros(2, 5, dtype=torch.int64))
        assert [(a.state, a.cache, a.attn_ws, a.n_splits) for a in model.layers] == held
