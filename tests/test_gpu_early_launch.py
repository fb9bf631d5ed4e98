"""Kernels that start while their predecessor on the stream ends read what it wrote.

Chains in which every call's inputs come from the call right before it, on buffers that hold another
input's values from the pass before: queued at once, and with the GPU waited for after each call.  Every
kernel here gives the same bits every run, so the two must agree to the last."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _norms(x, r, w, wait):
    import race_attention_b200 as rb
    y, h = wait(rb.add_rms_norm(x, r, w))
    rows = wait(rb.quant_int8(y))
    z = wait(rows.dequant(x.dtype))
    rows8, h2 = wait(rb.add_rms_norm_int8(z, h, w))
    v = wait(rows8.dequant(F32))
    y2, _ = wait(rb.add_rms_norm(v, None, v[-1]))  # the weight, too, was just written
    return y, h, rows.q, rows.scale, z, rows8.q, rows8.scale, h2, v, y2


def _products(x, r, w, wait):
    import race_attention_b200 as rb
    rows, _ = wait(rb.add_rms_norm_int8(x, r, w))
    out = []
    for tokens in (1, 20, 300, rows.q.shape[0]):  # the weights' rows and scales, too, were just written
        weights = wait(rb.quant_int8(r[:512]))
        y = wait(rb.int8_linear(rb.Int8Rows(rows.q[-tokens:], rows.scale[-tokens:]), weights, None, BF16))
        act = wait(rb.swiglu_int8(y))
        out += [y, act.q, act.scale, wait(act.dequant(BF16))]
    return out


def _log_probabilities(x, r, w, wait):
    import race_attention_b200 as rb
    logits, _ = wait(rb.add_rms_norm(x, r, w))
    leaf = logits.detach().requires_grad_(True)
    tokens = torch.arange(x.shape[0], device="cuda") * 7 % x.shape[1]
    res = wait(rb.token_logprobs(leaf, tokens, n_top=3))
    d, = wait(torch.autograd.grad((res.logp, res.entropy), leaf, (w[:1].expand(x.shape[0]).contiguous(), res.logp.detach())))
    rows = wait(rb.quant_int8(d))
    few = wait(rb.token_logprobs(d[-2:], tokens[-2:], n_top=5))
    return (*res, d, rows.q, rows.scale, *few)


def _gradients(x, r, w, wait):
    import race_attention_b200 as rb
    leaves = [t.detach().requires_grad_(True) for t in (x, r, w)]
    y, h = wait(rb.add_rms_norm(*leaves))
    dx, dr, dw = wait(torch.autograd.grad((y, h), leaves, (h.detach(), y.detach())))
    y2, h2 = wait(rb.add_rms_norm(dx, x, dw))  # dw: added up by the backward's last kernel
    return dx, dr, dw, y2, h2


@pytest.mark.parametrize("rows,K", [(2000, 1024), (5000, 2047), (30000, 256)])
@pytest.mark.parametrize("chain", [_norms, _products, _log_probabilities, _gradients])
def test_each_call_reads_what_the_one_before_it_wrote(chain, rows, K):
    g = torch.Generator(device="cuda").manual_seed(rows + K)
    inputs = [(torch.randn(rows, K, generator=g, device="cuda").to(BF16), torch.randn(rows, K, generator=g, device="cuda").to(BF16),
               torch.randn(K, generator=g, device="cuda")) for _ in range(3)]

    def synchronised(out):
        torch.cuda.synchronize()
        return out

    def leaves(out):
        return [t.detach().clone() for t in out if t is not None]

    want = [leaves(chain(*i, synchronised)) for i in inputs]
    for _ in range(3):
        for i, w in zip(inputs, want):
            got = chain(*i, lambda out: out)
            assert all(torch.equal(a, b) for a, b in zip(leaves(got), w, strict=True))
