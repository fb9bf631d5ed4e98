"""add_rms_norm, its gradient, and the 8-bit row operators against fp64 torch.

Tolerances: statistics are fp32 sums of at most 2^15 terms, of which no thread adds more than
1024 in a row, so a row's mean square is within 2^-14 of exact in the worst case and 1e-5 in
these; outputs are then rounded once to their type."""
import pytest
import torch

from _bounds import within

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5
STAT = 1e-5  # relative error of what is computed from a row's fp32 sums


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _near(got, want, dtype, scale=None, what=""):
    """got, of dtype, is the rounding of something within STAT of `scale` (default |want|) of want."""
    assert got.dtype == dtype
    want = want.double()
    # (and within the rounding of fp32 arithmetic after the sums: 2^-22 of the terms, under STAT)
    within(got, want, STAT * (want.abs() if scale is None else scale) + 1e-37, what)


def _norm64(x, r, w):
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    h64 = h.double()
    rstd = (h64.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return h, h64 * rstd * (1.0 if w is None else w.double()), rstd


SHAPES = [(1, 1), (1, 2048), (3, 7), (5, 64), (64, 2048), (33, 768), (17, 1000), (9, 2047), (7, 2056), (300, 4096),
          (2, 8192), (4, 8191), (3, 16384), (2, 32768), (2, 40001), (1500, 96)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,K", SHAPES)
def test_forward(rows, K, dtype):
    from race_attention_b200 import add_rms_norm
    g = _gen(rows * 7 + K)
    x, r = (torch.randn(rows, K, generator=g, device="cuda").to(dtype) for _ in range(2))
    for wt in (None, F32, BF16):
        w = None if wt is None else (1 + torch.randn(K, generator=g, device="cuda")).to(wt)
        for res in (None, r):
            h, want, _ = _norm64(x, res, w)
            y, got_h = add_rms_norm(x, res, w, eps=EPS)
            assert y.dtype == dtype and torch.equal(got_h, h)
            _near(y, want, dtype, what="y")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts_are_read_as_they_are(dtype):
    """Leading dimensions, row strides, odd starts, other orders and expanded rows."""
    from race_attention_b200 import add_rms_norm
    g = _gen(3)
    big = torch.randn(6, 5, 700, generator=g, device="cuda").to(dtype)
    cases = [big, big[:, :, :256], big[:, 1:3, 3:260], big[:, 2, 5:], big.transpose(0, 1), big.transpose(1, 2),
             big[:1, 0, :64].expand(4, 64), big[0, 0], big[..., ::2]]
    for x in cases:
        r = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
        h, want, _ = _norm64(x, r, None)
        y, got_h = add_rms_norm(x, r, None, eps=EPS)
        assert y.shape == x.shape and torch.equal(got_h, h)
        _near(y, want, dtype, what=str(x.stride()))
        y2, h2 = add_rms_norm(r, x, None, eps=EPS)
        assert torch.equal(y2, y) and torch.equal(h2, h)
    assert add_rms_norm(big[:0])[0].shape == (0, 5, 700)


def test_rows_that_are_not_finite_stay_alone():
    from race_attention_b200 import add_rms_norm, add_rms_norm_int8
    x = torch.randn(4, 300, generator=_gen(1), device="cuda")
    x[1, 17], x[2, 250] = float("nan"), float("inf")
    y, _ = add_rms_norm(x)
    rows, _ = add_rms_norm_int8(x)
    q = rows.dequant(F32)
    assert y[[0, 3]].isfinite().all() and q[[0, 3]].isfinite().all() and rows.scale[[0, 3]].isfinite().all()
    assert y[1].isnan().all() and y[2, 250].isnan() and not rows.scale[[1, 2]].isfinite().any()
    assert not q[[1, 2]].isfinite().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 2048), (5, 64), (64, 2048), (333, 768), (17, 1000), (9, 2047), (2, 8191),
                                    (2500, 96), (3, 16384), (2, 33000), (1201, 257)])
def test_gradient(rows, K, dtype):
    from race_attention_b200 import add_rms_norm
    g = _gen(rows + K)
    x, r, dy, dh = (torch.randn(rows, K, generator=g, device="cuda").to(dtype) for _ in range(4))
    for wt, res in ((F32, True), (BF16, True), (F32, False), (None, True)):
        w = None if wt is None else (1 + 0.3 * torch.randn(K, generator=g, device="cuda")).to(wt)
        leaves = [x.clone().requires_grad_(True)]
        if res:
            leaves.append(r.clone().requires_grad_(True))
        if w is not None:
            leaves.append(w.clone().requires_grad_(True))
        y, h = add_rms_norm(leaves[0], leaves[1] if res else None, None if w is None else leaves[-1], eps=EPS)
        outs, ups = ((y, h), (dy, dh)) if res else ((y,), (dy,))
        got = torch.autograd.grad(outs, leaves, ups)
        h64, _, rstd = _norm64(x, r if res else None, w)
        xh = h64.double() * rstd
        gg = dy.double() * (1.0 if w is None else w.double())
        c = (gg * xh).mean(-1, keepdim=True)
        cabs = (gg * xh).abs().mean(-1, keepdim=True)  # the fp32 sum's error goes by the terms' magnitudes
        dx = rstd * (gg - xh * c) + (dh.double() if res else 0)
        scale = rstd * (gg.abs() + xh.abs() * cabs) + (dh.double().abs() if res else 0)
        _near(got[0], dx, dtype, scale, "dx")
        if res:
            assert torch.equal(got[0], got[1])
        if w is not None:
            terms = dy.double() * xh
            _near(got[-1], terms.sum(0), wt, terms.abs().sum(0), "dw")


def test_gradient_against_differences():
    """d/dt of sum(a y + b h) along a random direction, by central differences of the fp32
    forward in a step of 2^-6: truncation and rounding are each under 1e-3 of the terms' sum."""
    from race_attention_b200 import add_rms_norm
    g = _gen(9)
    x, r, a, b, dx, dr = (torch.randn(6, 200, generator=g, device="cuda") for _ in range(6))
    w, dw = (1 + 0.3 * torch.randn(200, generator=g, device="cuda") for _ in range(2))

    def f(t):
        y, h = add_rms_norm(x + t * dx, r + t * dr, w + t * dw, eps=EPS)
        return float((a.double() * y.double()).sum() + (b.double() * h.double()).sum())

    leaves = [v.clone().requires_grad_(True) for v in (x, r, w)]
    grads = torch.autograd.grad(add_rms_norm(*leaves, eps=EPS), leaves, (a, b))
    slope = sum(float((u.double() * v.double()).sum()) for u, v in zip(grads, (dx, dr, dw)))
    step = 2.0 ** -6
    assert abs((f(step) - f(-step)) / (2 * step) - slope) < 1e-3 * float(a.abs().sum())


def test_gradient_of_one_output_alone_and_of_broadcast_weights():
    from race_attention_b200 import add_rms_norm
    g = _gen(4)
    x, r, dy = (torch.randn(2, 5, 160, generator=g, device="cuda") for _ in range(3))
    w = torch.ones(160, device="cuda", requires_grad=True)
    x1, r1 = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    y, h = add_rms_norm(x1, r1, w)
    gx, gr = torch.autograd.grad(h, (x1, r1), dy, retain_graph=True)
    assert torch.equal(gx, dy) and torch.equal(gr, dy)
    gx, gw = torch.autograd.grad(y, (x1, w), dy.transpose(0, 1).contiguous().transpose(0, 1), retain_graph=True)
    gx2, gw2 = torch.autograd.grad((y, h), (x1, w), (dy, torch.zeros_like(dy)))
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2)
    same = x.clone().requires_grad_(True)  # both terms the same tensor
    gs, = torch.autograd.grad(add_rms_norm(same, same, None)[0], same, dy)
    gd, = torch.autograd.grad(add_rms_norm(x1, x, None)[0], x1, dy)
    _near(gs, 2 * gd.double(), F32)


def test_gradient_bits_are_the_same_every_run():
    from race_attention_b200 import ops
    g = _gen(8)
    h, dy = (torch.randn(3000, 768, generator=g, device="cuda").to(BF16) for _ in range(2))
    w = torch.randn(768, generator=g, device="cuda")
    rstd = torch.rand(3000, generator=g, device="cuda") + 0.5
    first = ops.rms_norm_bwd(dy, None, h, rstd, w)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.rms_norm_bwd(dy, None, h, rstd, w)))


# ------------------------------------------------------------------- 8-bit rows
def _check_rows(rows, want, rel=STAT):
    """Each value within half a step (and the fp32 error of 127 steps) of the fp64 value."""
    want = want.double().reshape(-1, want.shape[-1])
    q, scale = rows.q.reshape(want.shape).double(), rows.scale.reshape(-1).double()
    amax = want.abs().amax(-1)
    assert bool(((scale - amax / 127).abs() <= rel * amax / 127 + 1e-44).all())
    assert bool((q.abs() <= 127).all()) and bool((q.abs().amax(-1) == torch.where(amax > 1e-40, 127.0, q.abs().amax(-1))).all())
    off = (q * scale[:, None] - want).abs()
    assert bool((off <= scale[:, None] * (0.5 + 2 * 127 * rel) + 1e-44).all()), float((off / scale[:, None]).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,K", SHAPES)
def test_int8_rows(rows, K, dtype):
    from race_attention_b200 import add_rms_norm_int8, quant_int8, swiglu_int8
    g = _gen(rows * 3 + K)
    x, r = (torch.randn(rows, K, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = 1 + torch.randn(K, generator=g, device="cuda")
    got = quant_int8(x)
    _check_rows(got, x)
    assert got.q.stride(0) % 16 == 0 or rows == 1
    # exact away from ties: the quotient's fp32 error is under 2^-16 of a step
    t = x.double() / got.scale.double()[:, None]
    sure = ((t - t.floor()) - 0.5).abs() > 2.0 ** -14
    assert bool((got.q.double() == t.round())[sure].all())
    _near(got.dequant(F32), got.q.double() * got.scale.double()[:, None], F32)
    _near(got.dequant(BF16), got.q.double() * got.scale.double()[:, None], BF16)
    for res in (None, r):
        h, want, _ = _norm64(x, res, w)
        got, got_h = add_rms_norm_int8(x, res, w, eps=EPS)
        assert torch.equal(got_h, h)
        _check_rows(got, want)
    gu = torch.randn(rows, 2 * K, generator=g, device="cuda").to(dtype) * 2
    gate, up = gu.double().chunk(2, -1)
    _check_rows(swiglu_int8(gu), gate * torch.sigmoid(gate) * up)


def _quotients(x):
    """Scales and 8-bit values by the definition: scale = max|x| times fp32's 1/127, the quotients
    rounded to fp32 as a division's are (from 64 bits: as many as that takes), then to whole numbers."""
    x = x.double()
    scale = (x.abs().amax(-1) * float(torch.tensor(1 / 127, dtype=F32))).to(F32)
    q = (x / scale.double()[..., None]).to(F32).round().clamp(-127, 127)
    return torch.where(scale[..., None] > 0, q, torch.zeros_like(q)).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,K", [(2000, 256), (64, 2048), (3000, 768), (700, 1000), (300, 2047), (100, 8192), (1500, 4096),
                                    (41, 8191), (20, 16384), (9, 40001)])
def test_int8_rows_are_the_quotients(rows, K, dtype):
    """Every value, those on half a step among them (which bf16 rows often hold): no tolerance."""
    from race_attention_b200 import quant_int8
    x = torch.randn(rows, K, generator=_gen(rows + 2 * K), device="cuda").to(dtype)
    x[0] = torch.arange(K, device="cuda") % 255 - 127  # halves and whole numbers of steps alone
    x[0, 0] = 63.5
    for v in (x, torch.cat([x, x], 1)[:, 1:K + 1]):
        got = quant_int8(v)
        q, scale = _quotients(v)
        assert torch.equal(got.scale, scale) and torch.equal(got.q, q)


@pytest.mark.parametrize("K", [96, 331, 2048, 40001])
def test_int8_rows_are_the_quotients_at_the_ends_of_the_range(K):
    from race_attention_b200 import quant_int8
    e = torch.arange(-149, 128, device="cuda", dtype=torch.float64)
    v = torch.randint(-255, 256, (277, K), generator=_gen(K), device="cuda").double() / 128
    x = (v * 2.0 ** e[:, None]).clamp(-3.3e38, 3.3e38).to(F32)
    got = quant_int8(x)
    q, scale = _quotients(x)
    assert torch.equal(got.scale, scale) and torch.equal(got.q, q)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,K,pad", [(1189, 2056, 0), (1187, 2048, 8), (1250, 4096, 16), (1190, 2048, 3), (1186, 2041, 7),
                                        (80003, 24, 0), (76802, 32, 8), (303107, 8, 8)])
def test_dequant_of_many_rows(rows, K, pad, dtype):
    # groups of rows that the last thread has only some of; row strides that are and are not whole words
    from race_attention_b200 import Int8Rows
    g = _gen(rows + K)
    q = torch.randint(-127, 128, (rows, K + pad), generator=g, device="cuda", dtype=torch.int8)[:, :K]
    scale = torch.rand(rows, generator=g, device="cuda") + 0.01
    got = Int8Rows(q, scale).dequant(dtype)
    assert got.shape == (rows, K) and got.dtype == dtype
    # one product in 32 bits, rounded once more for bf16
    assert torch.equal(got, (q.double() * scale.double()[:, None]).to(F32).to(dtype))


def test_int8_rows_of_zeros_tiny_and_huge_values():
    from race_attention_b200 import quant_int8
    x = torch.zeros(6, 100, device="cuda")
    x[1, 5] = 1e-38
    x[2] = torch.linspace(-1, 1, 100, device="cuda") * 3e38
    x[3] = torch.linspace(-1e-36, 1e-36, 100, device="cuda")
    x[4] = torch.linspace(-5e-40, 5e-40, 100, device="cuda")
    x[5, 99] = -7.0
    got = quant_int8(x)
    assert int(got.scale[0] != 0) == 0 and not got.q[0].any()
    assert bool(got.scale.isfinite().all())
    back = got.dequant(F32).double()
    # half a step, and the rounding of a step that is itself below the smallest normal number
    assert bool(((back - x.double()).abs() <= got.scale.double()[:, None] * 0.51 + 127 * 2.0 ** -149).all())
    assert int(got.q[5, 99]) == -127


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K", [64, 301, 2048, 20003])
def test_swiglu_of_gates_far_below_zero(K, dtype):
    """Gates whose e^-gate is near the end of fp32's range, times values that bring the products back:
    e^-|gate| is below the normal numbers, but by less than 2^-2, so it keeps 21 bits."""
    from race_attention_b200 import swiglu_int8
    g = _gen(K)
    gate = -87.4 - 1.2 * torch.rand(7, K, generator=g, device="cuda")
    up = torch.randn(7, K, generator=g, device="cuda") * 1e37
    gu = torch.cat([gate, up], 1).to(dtype)
    gate, up = gu.double().chunk(2, -1)
    _check_rows(swiglu_int8(gu), gate * torch.sigmoid(gate) * up)
    ends = torch.tensor([[-200.0, -1e30, 0.0, -0.0, 30.0, 1e30, -20.0, 1.0] + [1.0] * 8], device="cuda").to(dtype)
    gate, up = ends.double().chunk(2, -1)
    _check_rows(swiglu_int8(ends), gate * torch.sigmoid(gate) * up)


def test_int8_layouts():
    from race_attention_b200 import quant_int8, swiglu_int8
    g = _gen(5)
    big = torch.randn(6, 5, 702, generator=g, device="cuda")
    for x in (big, big[:, 1:3, 3:260], big[:, :, 5:], big.transpose(0, 1), big.transpose(1, 2), big[0, 0],
              big[:1, 0, :64].expand(4, 64)):
        rows = quant_int8(x)
        assert rows.shape == x.shape and rows.scale.shape == x.shape[:-1]
        _check_rows(rows, x)
    _check_rows(swiglu_int8(big[:, 2, 1:701]), (lambda a: torch.nn.functional.silu(a[:, :350]) * a[:, 350:])(big[:, 2, 1:701].double()))
    assert quant_int8(big[:0]).q.shape == (0, 5, 702)


def test_rows_past_two_gigabytes():
    """More than 2^31 values: the last rows, of aligned and of odd widths."""
    from race_attention_b200 import add_rms_norm, add_rms_norm_int8, ops
    g = _gen(14)
    for rows, K in ((1_100_000, 2048), (1_150_001, 2047)):
        x = torch.zeros(rows, K, device="cuda", dtype=BF16)
        x[:2] = torch.randn(2, K, generator=g, device="cuda").to(BF16)
        x[-9:] = torch.randn(9, K, generator=g, device="cuda").to(BF16)
        ends = [0, 1] + list(range(rows - 9, rows))
        y, h = add_rms_norm(x, x, None, eps=EPS)
        want_h, want, rstd = _norm64(x[ends], x[ends], None)
        assert torch.equal(h[ends], want_h)
        _near(y[ends], want, BF16, what="y")
        r8, _ = add_rms_norm_int8(x, None, None, eps=EPS)
        _check_rows(type(r8)(r8.q[ends], r8.scale[ends]), _norm64(x[ends], None, None)[1])
        dx, _ = ops.rms_norm_bwd(y, None, x, torch.ones(rows, device="cuda"), None, weight_grad=False)
        xs, ys = x[ends].double(), y[ends].double()
        c = (ys * xs).mean(-1, keepdim=True)
        cabs = (ys * xs).abs().mean(-1, keepdim=True)
        _near(dx[ends], ys - xs * c, BF16, ys.abs() + xs.abs() * cabs, "dx")
        del x, y, h, r8, dx


def test_runs_on_the_current_stream():
    """Inputs written on a side stream just before the call, on that stream."""
    from race_attention_b200 import add_rms_norm
    s = torch.cuda.Stream()
    x = torch.zeros(2000, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        x.fill_(2.0)
        y, _ = add_rms_norm(x, eps=0.0)
    s.synchronize()
    assert bool((y == 1.0).all())


def test_refusals():
    from race_attention_b200 import add_rms_norm, ops, quant_int8, swiglu_int8
    x = torch.zeros(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="dtype"):
        add_rms_norm(x.half())
    with pytest.raises(RuntimeError, match="shape and dtype"):
        add_rms_norm(x, x[:2])
    with pytest.raises(RuntimeError, match="shape and dtype"):
        add_rms_norm(x, x.bfloat16())
    with pytest.raises(RuntimeError, match="weight"):
        add_rms_norm(x, weight=torch.ones(65, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA only"):
        add_rms_norm(x.cpu())
    with pytest.raises(RuntimeError, match="CUDA only"):
        add_rms_norm(x, weight=torch.ones(64))
    with pytest.raises(RuntimeError, match="at least one value"):
        quant_int8(x[:, :0])
    with pytest.raises(RuntimeError, match="even"):
        swiglu_int8(x[:, :63])
    with pytest.raises(RuntimeError, match="rstd"):
        ops.rms_norm_bwd(x, None, x, torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="h's shape"):
        ops.rms_norm_bwd(x[:2], None, x, torch.ones(4, device="cuda"))
