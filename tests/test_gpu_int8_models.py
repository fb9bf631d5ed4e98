"""The 8-bit hybrid decoder and the log probabilities it answers with, and the GPT harness on the
fused norms and loss."""
import copy

import pytest
import torch

from conftest import relerr

pytestmark = pytest.mark.gpu


def _hybrid(seed=0):
    from race_attention_b200.hybrid import HybridConfig, HybridLlama
    torch.manual_seed(seed)
    cfg = HybridConfig(vocab_size=1000, n_layer=4, hidden=256, n_head=4, n_kv_head=2, mlp_hidden=512)
    model = HybridLlama(cfg).cuda()
    model.init_weights(0.05)
    return cfg, model.to(torch.bfloat16)


def _dequantised(model):
    """A float32 copy whose weights are the values the 8-bit rows stand for."""
    ref = copy.deepcopy(model).float()
    head = None
    for layer in ref.layers:
        for name in ("qkv", "o", "gate_up", "down"):
            w = getattr(layer, name).weight
            rows = __import__("race_attention_b200").quant_int8(w.to(torch.bfloat16))
            w.data.copy_(rows.dequant(torch.float32))
    return ref


def test_int8_decoder_is_near_its_float_form():
    """Weights as the 8-bit values stand for, so that only the activations' 8-bit steps (half a step
    of 1/127 of a row's largest value each, independent) and bf16 differ: the logits' error stays
    under 5% of their norm over four layers, step by step and from a prefill alike."""
    cfg, model = _hybrid()
    ref = _dequantised(model)
    model.quantize_int8()
    assert not any(isinstance(m, torch.nn.Linear) for m in model.modules())
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(0, cfg.vocab_size, (3, 150), device="cuda", generator=g)
    tok = model.prefill(idx, t_max=160, micro_batch=2)
    seq = idx
    for _ in range(4):
        seq = torch.cat([seq, tok[:, None]], 1)
        step = model.step_logits(tok).double()
        full = model.logits_full(seq).double()
        want = ref.logits_full(seq).double()
        assert float((step - want).norm() / want.norm()) < 0.05
        assert float((full - want).norm() / want.norm()) < 0.05
        tok = want.argmax(-1)
    assert model.n_tokens == 154


def test_int8_decode_graph_replays_the_eager_steps():
    from race_attention_b200.hybrid import DecodeGraph
    models = [_hybrid()[1].quantize_int8() for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(2)
    idx = torch.randint(0, 1000, (2, 100), device="cuda", generator=g)
    ta, tb = (m.prefill(idx, t_max=110) for m in models)
    assert torch.equal(ta, tb)
    ta, tb = (m.step(t) for m, t in zip(models, (ta, tb)))
    dg = DecodeGraph(models[1], tb)
    for _ in range(6):
        ta = models[0].step(ta)
        tb = dg.replay()
        assert torch.equal(ta, tb)


def test_quantising_twice_changes_nothing():
    _, model = _hybrid()
    model.quantize_int8()
    before = [m for m in model.modules()]
    held = {k: v.clone() for k, v in model.state_dict().items()}
    assert model.quantize_int8() is model
    assert all(a is b for a, b in zip(before, model.modules(), strict=True))
    assert all(torch.equal(held[k], v) for k, v in model.state_dict().items())


@pytest.mark.parametrize("int8", [False, True])
def test_answers_with_log_probabilities(int8):
    cfg, model = _hybrid(3)
    if int8:
        model.quantize_int8()
    g = torch.Generator(device="cuda").manual_seed(4)
    idx = torch.randint(0, cfg.vocab_size, (2, 60), device="cuda", generator=g)
    full = copy.deepcopy(model)
    tok = model.prefill(idx, t_max=64)
    nxt, lp = model.step_logprobs(tok, n_top=5)
    logits = full.logits_full(torch.cat([idx, tok[:, None]], 1)).double()
    assert torch.equal(lp.top_ids[:, 0], nxt) and torch.equal(lp.top_logp[:, 0], lp.logp)
    assert bool((lp.top_logp[:, :-1] >= lp.top_logp[:, 1:]).all())
    assert relerr(lp.logp, logits.log_softmax(-1).gather(-1, nxt[:, None])[:, 0]) < 5e-2
    # scores of a sequence: chunked or not, and against its own last logits
    s = full.score(idx, n_top=3)
    c = full.score(idx, n_top=3, positions=17)
    assert s.logp.shape == (2, 59) and s.top_ids.shape == (2, 59, 3)
    assert torch.allclose(s.logp, c.logp, atol=2e-2) and torch.allclose(s.entropy, c.entropy, atol=2e-2)
    last = full.logits_full(idx[:, :-1]).double().log_softmax(-1).gather(-1, idx[:, -1:])[:, 0]
    assert bool(((s.logp[:, -1].double() - last).abs() < 0.05 * last.abs()).all())
    assert full.pos is None  # scoring keeps no decode state
    one = full.score(idx[:, :1], n_top=2)  # nothing to score in a single token
    assert one.logp.shape == (2, 0) and one.top_ids.shape == (2, 0, 2)


def _gpt(fused):
    from race_attention_b200.gpt import GPTConfig, RaceGPT
    torch.manual_seed(0)
    cfg = GPTConfig(vocab_size=509, n_layer=2, n_head=2, n_embd=128, mlp_hidden=256, race_L=8, fused=fused)
    model = RaceGPT(cfg).cuda()
    model.init_weights(0.05)
    return cfg, model


def test_gpt_fused_matches_the_plain_harness():
    """The same weights through the fused norms and loss: bf16 activations, so loss and gradients
    agree within the bf16 tolerance of the harness (rel 2e-2 and, by 2-norm, 5e-2)."""
    cfg, plain = _gpt(False)
    _, fused = _gpt(True)
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(0, cfg.vocab_size, (2, 300), device="cuda", generator=g)
    tgt = torch.roll(idx, -1, 1)
    tgt[:, -1] = -100
    a, b = plain(idx, tgt), fused(idx, tgt)
    a.backward()
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) < 2e-2 * abs(float(a.detach()))
    for (name, p), q in zip(plain.named_parameters(), fused.parameters()):
        err = float((p.grad - q.grad).norm() / p.grad.norm())
        assert err < 5e-2, (name, err)


@pytest.mark.parametrize("norm_eps", [None, 1e-6, 1e-2])
def test_gpt_fused_norms_take_the_plain_ones_eps(norm_eps):
    """A residual stream whose mean square is near the smaller of these eps, one block and the whole model:
    both forms agree within the bf16 tolerance (5e-2 by 2-norm), where another eps is 20 % off or more."""
    from race_attention_b200.gpt import GPTConfig, RaceGPT
    outs = []
    for fused in (False, True):
        torch.manual_seed(0)
        cfg = GPTConfig(vocab_size=509, n_layer=2, n_head=2, n_embd=128, mlp_hidden=256, race_L=8, fused=fused,
                        norm_eps=norm_eps)
        model = RaceGPT(cfg).cuda()
        model.init_weights(0.05)
        g = torch.Generator(device="cuda").manual_seed(5)
        x = (torch.randn(1, 200, 128, device="cuda", generator=g) * 1e-3).bfloat16()
        idx = torch.randint(0, 509, (1, 200), device="cuda", generator=g)
        with torch.no_grad():
            cos, sin = model._angles(200, x.device, x.dtype)
            if fused:
                d, h = model.blocks[0].forward_fused(None, x, cos, sin)
                y = d.float() + h.float()
            else:
                y = model.blocks[0](x, cos, sin).float()
            model.wte.weight.mul_(0.02)
            outs.append((y, model(idx).float()))
    for a, b in zip(*outs):
        assert float((a - b).norm() / a.norm()) < 5e-2


def test_gpt_policy_gradient_steps():
    """A few steps on log probabilities weighted by advantages with an entropy bonus: the sampled
    tokens with positive advantages become more probable than those with negative ones."""
    cfg, model = _gpt(True)
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    g = torch.Generator(device="cuda").manual_seed(2)
    idx = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda", generator=g)
    tgt = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda", generator=g)
    adv = torch.where(torch.rand(2, 200, device="cuda", generator=g) < 0.5, 1.0, -0.2)
    gaps = []
    for _ in range(8):
        lp = model.token_logprobs(idx, tgt, n_top=2)
        gaps.append(float((lp.logp.detach()[adv > 0]).mean() - (lp.logp.detach()[adv < 0]).mean()))
        loss = -(adv * lp.logp).mean() - 1e-3 * lp.entropy.mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        assert all(p.grad.isfinite().all() for p in model.parameters() if p.grad is not None)
        opt.step()
    assert gaps[-1] > gaps[0] + 0.3, gaps
