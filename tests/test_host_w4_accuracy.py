"""The accuracy of 4-bit products without a GPU: the terms of an activation, and that the root-mean-square limits which the GPU
tests hold the kernels to are tight enough to tell three terms from two."""
import pytest
import torch

from oracle import few_token as ft

BF, FP = torch.bfloat16, torch.float16


def _w4(pkg, g, rows, cols, group, dt):
    w = pkg.ops.kernels.quantize_weight_int4((torch.randn((rows, cols), generator=g) * cols ** -0.5).to(dt), group)
    return w, ft.unpack(*w)


@pytest.mark.parametrize("dt,bits", [(BF, 23), (FP, 20)])
def test_three_terms_carry_every_value_of_the_type(dt, bits):
    """All finite values next to a largest one: exact down to 2^-bits of it, off by at most 2^-31 of it below."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dt).double()
    every = every[torch.isfinite(every)]
    for largest in (1.0, 1.9921875, 2.0 ** 15, 2.0 ** -10):
        v = every[every.abs() <= largest]
        x = torch.cat([torch.tensor([largest], dtype=torch.float64), v, torch.zeros(-(1 + len(v)) % 32)])
        got = ft.as_terms(x.expand(5, -1), 32)[0]
        near = x.abs() >= largest * 2.0 ** -bits
        assert torch.equal(got[near], x[near])
        assert (got - x).abs().max() <= largest * ft.TERM_FLOOR


@pytest.mark.parametrize("M,dt,group", [(4, BF, 128), (17, FP, 32), (64, BF, 64), (5, FP, 128)])
@pytest.mark.parametrize("outlier", [0.0, 1024.0, 16384.0])
def test_limits_tell_three_terms_from_two(pkg, M, dt, group, outlier):
    """Two terms carry 7 bits, which costs a bf16 value up to half of its last of 8 bits: about 2^-8.5 of the 64 scale
    steps times 2.9 that 4096 normal activations make, 0.5 steps. The limit is 300 * 2^-23 of the activations' length: 0.002
    steps without an outlier, 0.04 with 1024, 0.6 with 16384, where sums in 32 bits themselves hide the difference."""
    g = torch.Generator().manual_seed(M)
    w, full = _w4(pkg, g, 1024, 4096, group, dt)
    x = torch.randn((M, 4096), generator=g)
    if outlier:
        x[:, 77] = outlier
    x = x.to(dt).double()
    y = x @ full.t()
    rows = full[:, 77] == 0 if outlier else torch.ones(1024, dtype=torch.bool)
    res = ft.cancelling_residual(y, dt)
    limit = ft.product_rms_limit(x, w.scale, y[:, rows])
    for terms in (3, 2):
        got = (ft.as_terms(x, group, terms) @ full.t() + res.double()).to(dt)
        if terms == 3:
            ft.check_rms(got, y, res, limit, dt, "three terms", rows)
        elif outlier <= 1024:
            with pytest.raises(AssertionError, match="root-mean-square"):
                ft.check_rms(got, y, res, limit, dt, "two terms", rows)
