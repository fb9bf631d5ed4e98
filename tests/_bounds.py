"""Comparison of rounded outputs with 64-bit values."""


def within(got, want, slack, what=""):
    """Each entry of got is what some value within `slack` of `want` (both fp64) rounds to in got's
    type: rounding is monotone, so it lies between the roundings of want - slack and want + slack."""
    lo, hi = (want - slack).to(got.dtype).double(), (want + slack).to(got.dtype).double()
    g = got.double()
    ok = (lo <= g) & (g <= hi)
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} off, by up to {float((g - want).abs()[~ok].max())}"
