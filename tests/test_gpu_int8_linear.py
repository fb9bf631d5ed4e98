"""int8_linear against exact integer sums.

Tolerance: the sum is exact; its conversion to fp32, the two scales and the bias round four
times (2^-24 of the product, and of the bias), then outputs round once to their type."""
import pytest
import torch

from _bounds import within

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, rows, K, lo=-127, hi=127, pad=True):
    stride = -(-K // 16) * 16 if pad else K
    q = torch.empty(rows, stride, dtype=torch.int8, device="cuda")[:, :K]
    q.copy_(torch.randint(lo, hi + 1, (rows, K), generator=g, device="cuda", dtype=torch.int8))
    return q, torch.rand(rows, generator=g, device="cuda") * 0.02 + 1e-4


def _check(y, xq, xs, wq, ws, bias, dtype):
    acc = (xq.double() @ wq.double().t()) if xq.shape[-1] else 0  # below 2^53: exact
    prod = acc * xs.double()[:, None] * ws.double()
    want = prod if bias is None else prod + bias.double()
    assert y.dtype == dtype
    within(y, want, 2.0 ** -24 * 4 * (prod.abs() + (0 if bias is None else bias.double().abs())) + 1e-37)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 520])
@pytest.mark.parametrize("N,K", [(1, 1), (7, 16), (128, 128), (200, 130), (129, 2048), (2048, 513), (1000, 2050),
                                 (256, 4112), (4100, 64), (16, 8192)])
def test_shapes(M, N, K):
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(M * 31 + N * 7 + K)
    xq, xs = _rows(g, M, K)
    wq, ws = _rows(g, N, K)
    for dtype in (F32, BF16):
        for bias in (None, torch.randn(N, generator=g, device="cuda")):
            _check(int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws), bias, dtype), xq, xs, wq, ws, bias, dtype)


@pytest.mark.parametrize("M,N,K", [(2048, 2048, 512), (1111, 3001, 300), (4096, 256, 2048), (700, 20000, 256),
                                   (64, 16384, 2048), (9000, 129, 100)])
def test_large(M, N, K):
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(M + N + K)
    xq, xs = _rows(g, M, K)
    wq, ws = _rows(g, N, K)
    bias = torch.randn(N, generator=g, device="cuda")
    for dtype in (F32, BF16):
        _check(int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws), bias, dtype), xq, xs, wq, ws, bias, dtype)


@pytest.mark.parametrize("M", [3, 130, 300])
def test_largest_sums_do_not_overflow(M):
    from race_attention_b200 import Int8Rows, int8_linear
    K = 131071
    xq = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    wq = torch.full((5, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    wq[3:] = 127
    one = torch.ones(M, device="cuda")
    y = int8_linear(Int8Rows(xq, one), Int8Rows(wq, torch.ones(5, device="cuda")), None, F32)
    assert bool((y[:, :3] == float(16384 * K)).all()) and bool((y[:, 3:] == float(-128 * 127 * K)).all())


def test_layouts():
    """Leading dimensions; padded, wider, unpadded, shifted and transposed rows; strided scales."""
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(2)
    big = torch.randint(-127, 128, (40, 16, 96), generator=g, device="cuda", dtype=torch.int8)
    wide = torch.randint(-127, 128, (50, 200), generator=g, device="cuda", dtype=torch.int8)
    scale2 = torch.rand(50, 2, generator=g, device="cuda")
    for x in (big, big[:, 3], big[:, :, :80], big[0], big[:, 2, 1:81], big[:, 5, ::2][:, :40], big.transpose(0, 1), big[0, 0]):
        K = x.shape[-1]
        xs = torch.rand(x.shape[:-1], generator=g, device="cuda")
        for w in (wide[:, :K], wide[:, 16:16 + K], wide[:, 7:7 + K], wide[:, :K].contiguous(), wide.t()[:K, :50].t()):
            y = int8_linear(Int8Rows(x, xs), Int8Rows(w, scale2[:, 1]), None, F32)
            assert y.shape == x.shape[:-1] + (50,)
            _check(y.reshape(-1, 50), x.reshape(-1, K), xs.reshape(-1), w, scale2[:, 1], None, F32)
    assert int8_linear(Int8Rows(big[:0], torch.ones(0, 16, device="cuda")), Int8Rows(wide[:, :96], scale2[:, 0])).shape == (0, 16, 50)


def test_scales_that_are_not_finite_stay_in_their_rows():
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(6)
    xq, xs = _rows(g, 70, 256)
    wq, ws = _rows(g, 90, 256)
    xs[3], xs[66], ws[89] = float("nan"), float("inf"), float("nan")
    y = int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws), None, F32)
    keep = [i for i in range(70) if i not in (3, 66)]
    assert bool(y[keep, :89].isfinite().all()) and bool(y[3].isnan().all()) and bool(y[:, 89].isnan().all())
    assert not bool(y[66, :89].isfinite().any())


def test_linear_layer_from_a_float_one():
    """Quantising weights and tokens to 8 bits: each value is within half a step of its own, so the
    sum of K products with independent errors is within 2% of its 2-norm."""
    from race_attention_b200 import Int8Linear
    torch.manual_seed(0)
    lin = torch.nn.Linear(512, 384, device="cuda", dtype=BF16)
    x = torch.randn(3, 20, 512, device="cuda", dtype=BF16)
    layer = Int8Linear.from_linear(lin)
    want = torch.nn.functional.linear(x.double(), lin.weight.double(), lin.bias.double())
    y = layer(x)
    assert y.shape == want.shape and y.dtype == BF16
    assert float((y.double() - want).detach().norm() / want.detach().norm()) < 0.02
    assert set(layer.state_dict()) == {"q", "scale", "bias"}


def test_linear_layer_of_odd_width_keeps_its_form_when_moved():
    from race_attention_b200 import Int8Linear
    torch.manual_seed(1)
    layer = Int8Linear(torch.randn(65, 77, device="cuda"), torch.randn(65, device="cuda"), F32)
    x = torch.randn(9, 77, device="cuda")
    y = layer(x)
    moved = layer.to(BF16).cpu().cuda()
    assert moved.scale.dtype == F32 and moved.bias.dtype == F32 and moved.q.dtype == torch.int8
    assert torch.equal(moved(x), y)
    other = Int8Linear(torch.zeros(65, 77, device="cuda"), torch.zeros(65, device="cuda"), F32)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)


@pytest.mark.parametrize("M,N", [(66000, 33000), (33000, 66001)])
def test_outputs_past_two_gigabytes(M, N):
    """More than 2^31 outputs: the last rows and columns are where they belong."""
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(31)
    xq, xs = _rows(g, M, 64)
    wq, ws = _rows(g, N, 64)
    y = int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws))
    for at in (slice(0, 2), slice(M - 300, M)):
        _check(y[at], xq[at], xs[at], wq, ws, None, BF16)


def test_other_stream_and_repeated_calls_give_the_same_bits():
    from race_attention_b200 import Int8Rows, int8_linear
    g = _gen(11)
    for M, N, K in ((1, 2048, 2048), (64, 4096, 2048), (300, 1000, 1024), (1500, 1500, 512)):
        xq, xs = _rows(g, M, K)
        wq, ws = _rows(g, N, K)
        first = int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            outs = [int8_linear(Int8Rows(xq, xs), Int8Rows(wq, ws)) for _ in range(5)]
        side.synchronize()
        assert all(torch.equal(first, o) for o in outs)


def test_expired_wait_is_reported():
    """With no tile loaded the first wait runs out: the call says so, its output is NaN, and the
    next call is right."""
    from race_attention_b200 import Int8Rows, _lib, int8_linear
    lib = _lib.load()
    g = _gen(12)
    for M, N, K in ((4, 300, 256), (700, 600, 256)):
        xq, xs = _rows(g, M, K)
        wq, ws = _rows(g, N, K)
        x, w = Int8Rows(xq, xs), Int8Rows(wq, ws)
        want = int8_linear(x, w, None, F32)
        out = None
        lib.race_set_wait_limit(20000)
        lib.race_test_withhold_first_load(1)
        lib.race_set_status_check(0)
        try:
            out = int8_linear(x, w, None, F32)
            torch.cuda.synchronize()
            lib.race_set_status_check(1)
            with pytest.raises(RuntimeError, match="wait"):
                int8_linear(x, w, None, F32)
        finally:
            lib.race_set_wait_limit(0)
            lib.race_test_withhold_first_load(0)
            lib.race_set_status_check(1)
        assert bool(out.isnan().all())
        assert torch.equal(int8_linear(x, w, None, F32), want)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 2048), (4, 300, 256), (33, 700, 4096), (64, 4096, 2048), (128, 2048, 8192),
                                   (300, 1000, 1024), (1500, 1500, 512), (2100, 3000, 3001), (9000, 700, 100)])
def test_waits_that_run_out_while_copies_are_under_way(M, N, K):
    """Limits of a few polls: waits give up early or late, with tile loads and products on their way, and
    once with no load at all.  Each output is NaN or right, and the next call is right: the kernel has
    waited for its copies and products and given its TMEM back."""
    from race_attention_b200 import Int8Rows, _lib, int8_linear
    lib = _lib.load()
    g = _gen(M + N + K + 1)
    x, w = Int8Rows(*_rows(g, M, K)), Int8Rows(*_rows(g, N, K))
    want = int8_linear(x, w, None, F32)
    gave_up = 0
    for polls, withhold in [(n, 0) for n in (1, 2, 4, 8, 16, 32, 64, 128, 256)] + [(64, 1)]:
        lib.race_set_wait_limit(polls)
        lib.race_test_withhold_first_load(withhold)
        lib.race_set_status_check(0)
        try:
            outs = [int8_linear(x, w, None, F32) for _ in range(3)]
            torch.cuda.synchronize()
        finally:
            lib.race_set_wait_limit(0)
            lib.race_test_withhold_first_load(0)
            lib.race_set_status_check(1)
        expired = any(bool(o.isnan().any()) for o in outs)
        gave_up += expired
        assert all(bool((o.isnan() | (o == want)).all()) for o in outs)
        if withhold:
            assert all(bool(o.isnan().all()) for o in outs)
        if expired:  # said once, by the next call that asks
            with pytest.raises(RuntimeError, match="wait"):
                int8_linear(x, w, None, F32)
        assert torch.equal(int8_linear(x, w, None, F32), want)
    assert gave_up


def test_refusals():
    from race_attention_b200 import Int8Rows, int8_linear
    q = torch.zeros(4, 64, dtype=torch.int8, device="cuda")
    s = torch.ones(4, device="cuda")
    x = Int8Rows(q, s)
    with pytest.raises(RuntimeError, match="int8"):
        int8_linear(Int8Rows(q.float(), s), x)
    with pytest.raises(RuntimeError, match="scales"):
        int8_linear(Int8Rows(q, s[:3]), x)
    with pytest.raises(RuntimeError, match="scales"):
        int8_linear(Int8Rows(q, s.double()), x)
    with pytest.raises(RuntimeError, match=r"\[N, 64\]"):
        int8_linear(x, Int8Rows(q[:, :32], s))
    with pytest.raises(RuntimeError, match="bias"):
        int8_linear(x, x, torch.ones(5, device="cuda"))
    with pytest.raises(RuntimeError, match="bias"):
        int8_linear(x, x, torch.ones(4, device="cuda", dtype=BF16))
    with pytest.raises(RuntimeError, match="dtype"):
        int8_linear(x, x, None, torch.float16)
    with pytest.raises(RuntimeError, match="CUDA only"):
        int8_linear(x, Int8Rows(q.cpu(), s))
    long = torch.zeros(2, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError, match="131071"):
        int8_linear(Int8Rows(long, s[:2]), Int8Rows(long, s[:2]))
