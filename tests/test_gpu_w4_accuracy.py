"""How exact the 4-bit products are: root-mean-square errors against limits that grow like the root of the columns (oracle/
few_token.py), with the output's own rounding cancelled by a residual, so that what is seen is the sums in 32 bits."""
import pytest
import torch

from oracle import few_token as ft

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rnd(g, *shape, std=1.0, dt=BF):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dt)


def _w4(pkg, g, *shape, group, symmetric=False, dt=BF):
    return pkg.ops.kernels.quantize_weight_int4(_rnd(g, *shape, std=shape[-1] ** -0.5, dt=dt), group, symmetric)


@pytest.mark.parametrize("M", [1, 4, 5, 16, 17, 64])
@pytest.mark.parametrize("dt,group", [(BF, 128), (FP, 128), (BF, 32), (FP, 64)])
@pytest.mark.parametrize("outlier", [1024.0, 16384.0])
def test_an_outlier_channel_costs_the_other_channels_nothing(pkg, cuda_dev, M, dt, group, outlier):
    """One activation of every token is some thousand times larger than the rest. Outputs whose weight on it is zero are
    as exact as the 32-bit sums they are made of, whether 4 or 5 tokens are in the call."""
    g = _gen(cuda_dev, M + group)
    w = _w4(pkg, g, 1500, 4096, group=group, dt=dt)
    full = ft.unpack(*w)
    x = _rnd(g, M, 4096, dt=dt)
    x[:, 77] = outlier
    y = x.double() @ full.t()
    rows = full[:, 77] == 0
    assert int(rows.sum()) > 100
    res = ft.cancelling_residual(y, dt)
    got = pkg.ops.kernels.linear_w4(x, w, residual=res)
    ft.check_rms(got, y, res, ft.product_rms_limit(x.double(), w.scale, y[:, rows]), dt, f"M={M} g{group} {outlier}", rows)
    ft.check_rms(got, y, res, ft.product_rms_limit(x.double(), w.scale, y), dt, f"M={M} g{group} {outlier}, all rows")


@pytest.mark.parametrize("M", [1, 5, 33])
@pytest.mark.parametrize("up", [90, -100])
def test_scales_and_activations_at_opposite_ends_of_bfloat16(pkg, cuda_dev, M, up):
    """Scales around 2^90 (2^-100) times activations around 2^-60 (2^60): products in the middle of the type."""
    g = _gen(cuda_dev, M)
    w = _w4(pkg, g, 300, 4096, group=64)
    w = w._replace(scale=(w.scale.double() * 2.0 ** up).to(BF))
    x = (_rnd(g, M, 4096).double() * 2.0 ** (-60 if up > 0 else 60)).to(BF)
    y = pkg.ops.kernels.linear_w4(x, w)
    ft.check(y, *ft.linear(x, ft.unpack(*w), None, None, BF, 64), f"M={M} 2^{up}")
    want = x.double() @ ft.unpack(*w).t()
    assert (ft.rms(y.double() - want) <= ft.product_rms_limit(x.double(), w.scale, want, torch.finfo(BF).eps / 2)).all()
