"""token_logprobs and its gradient against fp64 torch.

Tolerances: z = logit / temperature rounds once (2^-24 |z|, |z| < 64 here), each exp is within
2^-21 + 2^-24 |z - max| of itself and the sums are fp32 of at most 2^12 terms in a row, so lse is
within 2e-5 and so are logp and the entropy (whose terms carry |z - lse| < 64: 1e-4).  A gradient
is p (or 1 - p) times its upstream: within 1e-4 of the terms, and its own rounding."""
import math

import pytest
import torch

from _bounds import within

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NEG = -math.inf


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _reference(logits, tokens, temperature, n_top, ignore=-100):
    z = logits.double() / temperature
    lse = torch.logsumexp(z, -1, keepdim=True)
    logq = torch.where(lse == NEG, torch.full_like(z, NEG), z - lse)
    p = logq.exp()
    entropy = -torch.where(p > 0, p * logq, torch.zeros_like(p)).sum(-1)
    used = tokens != ignore
    logp = logq.gather(-1, tokens.clamp(0, logits.shape[-1] - 1)[..., None])[..., 0]
    order = torch.sort(logits.double() + 0.0, dim=-1, descending=True, stable=True).indices[..., :n_top]
    top = logq.gather(-1, order)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    return (torch.where(used, logp, zero), torch.where(used, entropy, zero), torch.where(used[..., None], order, -1),
            torch.where(used[..., None], top, torch.full_like(top, NEG)), logq, p)


def _near(got, want, tol, what):
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    assert bool((off <= tol).all()), f"{what}: {float(off.max())}"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (1, 5, 5), (3, 31, 31), (4, 257, 20), (2, 1000, 32), (5, 4096, 0),
                                        (7, 8191, 5), (64, 12800, 20), (3, 50257, 32), (2, 131072, 7), (600, 777, 3),
                                        (400, 50257, 0), (2, 300000, 20), (200, 40000, 32)])
def test_forward(rows, V, top, dtype):
    from race_attention_b200 import token_logprobs
    g = _gen(rows * 5 + V)
    for temperature, scale in ((1.0, 2.5), (0.7, 6.0), (5.0, 1.0)):
        logits = (torch.randn(rows, V, generator=g, device="cuda") * scale).to(dtype)
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        if rows > 2:
            tokens[1] = -100
        logp, entropy, ids, top_logp, *_ = _reference(logits, tokens, temperature, top)
        got = token_logprobs(logits, tokens, temperature=temperature, n_top=top)
        _near(got.logp, logp, 2e-5, "logp")
        _near(got.entropy, entropy, 1e-4, "entropy")
        assert torch.equal(got.top_ids, ids)
        _near(got.top_logp, top_logp, 2e-5, "top_logp")


@pytest.mark.parametrize("V", [40, 1003, 33000])
def test_ties_go_to_the_lowest_index(V):
    from race_attention_b200 import token_logprobs
    g = _gen(V)
    tokens = torch.zeros(8, dtype=torch.int64, device="cuda")
    few = torch.randint(0, 3, (8, V), generator=g, device="cuda").float()      # three values only
    few[0] = 1.0                                                               # all alike
    few[1] = torch.where(torch.rand(V, generator=g, device="cuda") < 0.5, 0.0, -0.0)  # +-0 are alike
    few[2] = torch.arange(V, device="cuda") * 1e-3                             # the largest last
    few[3] = -few[2]                                                           # and first
    few[4] = NEG                                                               # fewer entries than alternatives
    few[4, V // 2], few[4, 3] = 1.0, 1.0
    few[5] = NEG
    few[5, V - 1] = -5.0
    few[6, ::2] = 2.5
    for dtype in (F32, BF16):
        logits = few.to(dtype)
        _, _, ids, top, *_ = _reference(logits, tokens, 1.0, 32)
        got = token_logprobs(logits, tokens, n_top=32)
        assert torch.equal(got.top_ids, ids)
        _near(got.top_logp, top, 2e-5, "top_logp")


@pytest.mark.parametrize("V,dtype", [(4000, BF16), (2000, F32), (3993, BF16), (2047, F32)])
def test_alternatives_of_many_random_rows(V, dtype):
    """About one such row in a hundred has more entries at or above the bound than are ranked at once."""
    from race_attention_b200 import token_logprobs
    g = _gen(V + 3)
    logits = torch.randn(4000, V, generator=g, device="cuda").to(dtype)
    tokens = torch.zeros(4000, dtype=torch.int64, device="cuda")
    _, _, ids, top, *_ = _reference(logits, tokens, 1.0, 32)
    got = token_logprobs(logits, tokens, n_top=32)
    assert torch.equal(got.top_ids, ids)
    _near(got.top_logp, top, 2e-5, "top_logp")


# rows, vocabulary of bf16 and fp32 rows, threads per block, blocks per row, entries ranked at once
@pytest.mark.parametrize("rows,Vs,threads,blocks,places", [
    (40, (4000, 2000), 32, 1, 256), (41, (2999, 2047), 32, 1, 256), (700, (10000, 8000), 128, 1, 1024),
    (33, (9999, 7999), 128, 1, 1024), (700, (40000, 20000), 256, 1, 1024), (601, (33001, 16501), 256, 1, 1024),
    (200, (65536, 32768), 256, 2, 1024), (3, (131072, 131072), 256, 8, 1024), (2, (200003, 160003), 256, 8, 1024)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_alternatives_that_lie_with_few_threads(rows, Vs, threads, blocks, places, dtype):
    """The large entries of each block's share are those of n_top - 1 threads (all of them: far more than
    are ranked at once), so the n_top-th thread's maximum, which bounds the alternatives, is low."""
    from race_attention_b200 import token_logprobs
    V, per = (Vs[1], 4) if dtype == F32 else (Vs[0], 8)
    g = _gen(rows + V)
    off = (torch.arange(rows, device="cuda") * V % per)[:, None]
    granules = (V + off + per - 1) // per
    granule = (torch.arange(V, device="cuda") + off) // per
    first = torch.zeros_like(granule)  # of the block's share that a granule is in
    for b in range(1, blocks):
        at = granules * b // blocks
        first = torch.where(granule >= at, at, first)
    thread = (granule - first) % threads
    for n in (32, 20):
        step = max(1, threads // 32)
        high = (thread % step == 0) & (thread // step < n - 1)
        for b in range(blocks):
            share = (granule >= granules * b // blocks) & (granule < granules * (b + 1) // blocks)
            assert int((high & share).sum(1).min()) > places
        x = torch.randn(rows, V, generator=g, device="cuda")
        logits = torch.where(high, 10 + x.abs() / 8, x.clamp(-3, 3)).to(dtype)
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        _, _, ids, top, *_ = _reference(logits, tokens, 1.0, n)
        for _ in range(2):
            got = token_logprobs(logits, tokens, n_top=n)
            assert torch.equal(got.top_ids, ids)
            _near(got.top_logp, top, 2e-5, "top_logp")


@pytest.mark.parametrize("V", [5, 700, 50257])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks_and_rows_without_an_entry(V, dtype):
    from race_attention_b200 import token_logprobs
    g = _gen(V + 1)
    logits = torch.randn(7, V, generator=g, device="cuda").to(dtype)
    logits[0, 1:] = NEG                              # one entry left
    logits[1] = NEG                                  # none
    logits[2, torch.rand(V, generator=g, device="cuda") < 0.9] = NEG
    logits[2, 0] = 0.5
    logits[3] = torch.finfo(dtype).min               # masked by the type's lowest value instead
    logits[3, 2] = 1.0
    logits[4, V // 2] = float("nan")
    logits[5, V - 1] = float("inf")
    tokens = torch.tensor([0, 1, 0, 2, 0, 1, 3], device="cuda")
    lg = logits.clone().requires_grad_(True)
    n = min(V, 4)
    got = token_logprobs(lg, tokens, n_top=n)
    d, = torch.autograd.grad((got.logp, got.entropy), lg, (torch.ones(7, device="cuda"), torch.ones(7, device="cuda")))
    logp, entropy, ids, top, logq, p = _reference(logits, tokens, 1.0, n)
    good = [0, 1, 2, 3, 6]
    _near(got.logp[good], logp[good], 2e-5, "logp")
    _near(got.entropy[good], entropy[good], 1e-4, "entropy")
    assert torch.equal(got.top_ids[good], ids[good])
    _near(got.top_logp[good], top[good], 2e-5, "top_logp")
    assert got.logp[0] == 0 and got.entropy[0] == 0 and got.logp[1] == NEG and got.entropy[1] == 0
    assert bool(got.logp[[4, 5]].isnan().all()) and bool(got.entropy[[4, 5]].isnan().all())
    assert int(got.top_ids[4].min()) >= 0 and V // 2 not in got.top_ids[4].tolist()[:n - 1] and int(got.top_ids[5, 0]) == V - 1
    assert bool(d[good].isfinite().all()) and not bool(d[1].any()) and bool((d[2][logits[2] == NEG] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [3, 1000, 70001])
def test_rows_of_the_lowest_value_alone_are_uniform(V, dtype):
    """A mask by the type's lowest value that leaves nothing: every entry is as probable."""
    from race_attention_b200 import token_logprobs
    logits = torch.full((3, V), torch.finfo(dtype).min, device="cuda", dtype=dtype, requires_grad=True)
    tokens = torch.tensor([0, V // 2, V - 1], device="cuda")
    got = token_logprobs(logits, tokens, n_top=2)
    want = torch.full((3,), -math.log(V), device="cuda")
    _near(got.logp, want, 2e-5, "logp")
    _near(got.entropy, -want, 1e-4, "entropy")
    assert torch.equal(got.top_ids.cpu(), torch.tensor([[0, 1]] * 3))
    d, = torch.autograd.grad(got.logp.sum(), logits)
    one = torch.zeros(3, V, device="cuda", dtype=torch.float64).scatter_(1, tokens[:, None], 1.0)
    within(d, one - 1 / V, 1e-4 * (one + 1 / V), "dlogits")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 9), (5, 257), (3, 1000), (33, 8191), (6, 50257), (2, 131072), (700, 640)])
def test_gradient(rows, V, dtype):
    from race_attention_b200 import token_logprobs
    g = _gen(rows + V)
    for temperature in (1.0, 0.7):
        logits = (torch.randn(rows, V, generator=g, device="cuda") * 2.5).to(dtype)
        tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
        if rows > 2:
            tokens[1] = -100
        a, b = (torch.randn(rows, generator=g, device="cuda") for _ in range(2))
        used = (tokens != -100).double()[:, None]
        _, entropy, _, _, logq, p = _reference(logits, tokens, temperature, 0)
        one = torch.zeros_like(p).scatter_(1, tokens.clamp(min=0)[:, None], 1.0)
        for ga, gb in ((a, b), (a, None), (None, b)):
            lg = logits.clone().requires_grad_(True)
            got = token_logprobs(lg, tokens, temperature=temperature)
            outs = [o for o, u in ((got.logp, ga), (got.entropy, gb)) if u is not None]
            d, = torch.autograd.grad(outs, lg, [u for u in (ga, gb) if u is not None])
            A = (torch.zeros_like(a) if ga is None else ga).double()[:, None] * used
            B = (torch.zeros_like(b) if gb is None else gb).double()[:, None] * used
            H = -(p * logq).sum(-1, keepdim=True)
            want = (A * (one - p) - B * p * (logq + H)) / temperature
            terms = (A.abs() * (one + p) + B.abs() * p * (logq.abs() + H)) / temperature
            assert d.dtype == dtype
            within(d, want, 1e-4 * terms + 1e-37, "dlogits")
            if rows > 2:
                assert not bool(d[1].any())


def test_gradient_against_differences():
    """Slope of sum(a logp + b entropy) along a random direction by central differences in a step
    of 2^-5: the third derivative of a row's terms is under 8, the forward's error under 2e-5, so
    the slope is within (8 step^2 / 6 + 2e-5 / step) of each row's |a| + |b|."""
    from race_attention_b200 import token_logprobs
    g = _gen(21)
    R, V, step = 6, 300, 2.0 ** -5
    x, d = (torch.randn(R, V, generator=g, device="cuda") for _ in range(2))
    a, b = (torch.randn(R, generator=g, device="cuda") for _ in range(2))
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")

    def f(t):
        r = token_logprobs(x + t * d, tokens)
        return float((a.double() * r.logp.double()).sum() + (b.double() * r.entropy.double()).sum())

    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, tokens)
    grad, = torch.autograd.grad((r.logp, r.entropy), leaf, (a, b))
    slope = float((grad.double() * d.double()).sum())
    bound = (8 * step * step / 6 + 2e-5 / step) * float((a.abs() + b.abs()).sum())
    assert abs((f(step) - f(-step)) / (2 * step) - slope) < bound


def test_entropies_are_not_negative():
    """Peaked rows, whose entropy is below the rounding of its terms."""
    from race_attention_b200 import token_logprobs
    g = _gen(26)
    logits = torch.randn(4000, 97, generator=g, device="cuda")
    logits[:, 3] += torch.linspace(5, 60, 4000, device="cuda")
    got = token_logprobs(logits, torch.full((4000,), 3, device="cuda"))
    assert bool((got.entropy >= 0).all()) and bool((got.logp <= 0).all())


def test_cross_entropy_is_the_mean_of_the_rest():
    from race_attention_b200 import token_logprobs
    g = _gen(22)
    logits = torch.randn(2, 50, 999, generator=g, device="cuda")
    tokens = torch.randint(0, 999, (2, 50), generator=g, device="cuda")
    tokens[0, 3:9] = -100
    l1, l2 = logits.clone().requires_grad_(True), logits.double().requires_grad_(True)
    loss = -token_logprobs(l1, tokens).logp.sum() / (tokens != -100).sum()
    want = torch.nn.functional.cross_entropy(l2.flatten(0, 1), tokens.flatten())
    loss.backward()
    want.backward()
    _near(loss, want, 2e-5, "loss")
    _near(l1.grad, l2.grad, 1e-4 / 94, "gradient")


def test_layouts_and_other_ignore_index():
    from race_attention_b200 import token_logprobs
    g = _gen(23)
    for dtype in (F32, BF16):
        big = (torch.randn(6, 5, 1301, generator=g, device="cuda") * 2).to(dtype)
        for x in (big, big[:, :, :1280], big[:, 1:3, 3:1000], big[:, 2, 5:], big.transpose(0, 1), big.transpose(1, 2),
                  big[0, 0], big[:1, 0, :64].expand(4, 64)):
            V = x.shape[-1]
            tokens = torch.randint(0, V, x.shape[:-1], generator=g, device="cuda")
            if tokens.dim():
                tokens[0] = 3
            logp, entropy, ids, top, logq, p = _reference(x, tokens, 1.0, 4)
            leaf = x.detach().requires_grad_(True)
            got = token_logprobs(leaf, tokens, n_top=4, ignore_index=1 << 40)
            _near(got.logp, logp, 2e-5, "logp")
            _near(got.entropy, entropy, 1e-4, "entropy")
            assert torch.equal(got.top_ids, ids)
            d, = torch.autograd.grad(got.logp.sum(), leaf)
            one = torch.zeros_like(p).scatter_(-1, tokens[..., None], 1.0)
            within(d, one - p, 1e-4 * (one + p), "dlogits")
            if tokens.dim():
                same = token_logprobs(x, tokens, n_top=4, ignore_index=3)
                assert not bool(same.logp[0].any()) and bool((same.top_ids[0] == -1).all())
    assert token_logprobs(big[:0, 0], tokens.new_zeros(0), n_top=2).top_ids.shape == (0, 2)


def test_tokens_outside_the_vocabulary_give_nan():
    from race_attention_b200 import token_logprobs
    logits = torch.randn(4, 100, generator=_gen(24), device="cuda", requires_grad=True)
    tokens = torch.tensor([100, -1, 1 << 40, 5], device="cuda")
    got = token_logprobs(logits, tokens, n_top=2)
    assert bool(got.logp[:3].isnan().all()) and bool(got.logp[3].isfinite()) and bool(got.entropy.isfinite().all())
    d, = torch.autograd.grad(got.logp.sum(), logits)
    assert bool(d[:3].isnan().all()) and bool(d[3].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [100, 1001, 33000])
def test_tokens_outside_the_vocabulary_leave_other_gradients_alone(V, dtype):
    """Rows whose log probability is not used (masked out, or the entropy alone taken) have the
    gradients that any token gives them."""
    from race_attention_b200 import token_logprobs
    g = _gen(V + 27)
    x = torch.randn(4, V, generator=g, device="cuda").to(dtype)
    bad = torch.tensor([V, -1, 1 << 40, 5], device="cuda")
    good = torch.tensor([1, 2, 3, 5], device="cuda")
    w = torch.randn(4, generator=g, device="cuda")
    got = []
    for tokens in (bad, good):
        for view in (x, torch.cat([x, x], 1)[:, 3:3 + V]):  # rows like the gradient's, and not
            leaf = view.detach().requires_grad_(True)
            r = token_logprobs(leaf, tokens)
            kept = torch.where(bad == good, r.logp, torch.zeros_like(r.logp))
            got.append([torch.autograd.grad(out, leaf, retain_graph=True)[0]
                        for out in ((w * r.entropy).sum(), (kept * w).sum(), (kept * w).sum() + (w * r.entropy).sum())])
    for a, b in zip(got[:2], got[2:]):
        for da, db in zip(a, b):
            assert bool(da.isfinite().all()) and torch.equal(da, db)
        assert not bool(a[1][:3].any())


def test_rows_past_two_gigabytes():
    """Offsets past 2^31 elements and 2^32 bytes: the last rows of a long batch."""
    from race_attention_b200 import token_logprobs
    rows, V = 17000, 131072
    logits = torch.zeros(rows, V, device="cuda", dtype=BF16)
    g = _gen(25)
    logits[-2:] = torch.randn(2, V, generator=g, device="cuda").to(BF16)
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
    leaf = logits.requires_grad_(True)
    got = token_logprobs(leaf, tokens, n_top=2)
    logp, entropy, ids, *_, p = _reference(logits[-2:].detach(), tokens[-2:], 1.0, 2)
    _near(got.logp[-2:], logp, 2e-5, "logp")
    assert torch.equal(got.top_ids[-2:], ids) and torch.equal(got.top_ids[:3].cpu(), torch.tensor([[0, 1]] * 3))
    _near(got.logp[:1], torch.tensor([-math.log(V)], device="cuda"), 2e-5, "uniform")
    d, = torch.autograd.grad(got.logp[-1], leaf)
    one = torch.zeros_like(p[-1]).index_fill_(0, tokens[-1], 1.0)
    within(d[-1], one - p[-1], 1e-4 * (one + p[-1]), "dlogits")
    assert not bool(d[-2].any())


def test_refusals():
    from race_attention_b200 import token_logprobs
    x = torch.zeros(4, 64, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(RuntimeError, match="int64"):
        token_logprobs(x, t[:3])
    with pytest.raises(RuntimeError, match="dtype"):
        token_logprobs(x.half(), t)
    with pytest.raises(RuntimeError, match="CUDA only"):
        token_logprobs(x, t.cpu())
    for n in (-1, 33, 65):
        with pytest.raises(RuntimeError, match="alternatives"):
            token_logprobs(torch.zeros(4, 64, device="cuda"), t, n_top=n)
    with pytest.raises(RuntimeError, match="alternatives"):
        token_logprobs(x[:, :3], t, n_top=4)
    for temp in (0.0, -1.0, math.inf, math.nan, 1e-39):
        with pytest.raises(RuntimeError, match="temperature"):
            token_logprobs(x, t, temperature=temp)
