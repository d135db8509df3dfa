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


@pytest.mark.parametrize("M", [1, 3, 4, 5, 8, 16, 17, 33, 64])
@pytest.mark.parametrize("dt,group", [(BF, 128), (FP, 32)])
def test_linear_with_many_units_per_block(pkg, cuda_dev, M, dt, group):
    """Every ring of the stream kernel turns several times (about 14 units of 65,536 weights per block): stale or mixed-up
    terms, factors or scales would be far outside."""
    g = _gen(cuda_dev, M)
    w = _w4(pkg, g, 16384, 8192, group=group, symmetric=M == 8, dt=dt)
    x = _rnd(g, M, 8192, dt=dt)
    y = x.double() @ ft.unpack(*w).t()
    res = ft.cancelling_residual(y, dt)
    got = pkg.ops.kernels.linear_w4(x, w, residual=res)
    ft.check_rms(got, y, res, ft.product_rms_limit(x.double(), w.scale, y), dt, f"M={M} g{group}")


@pytest.mark.parametrize("M,K,N,group,act,bias,dt", [
    (1, 4096, 14336, 128, "silu", False, BF), (4, 4096, 6144, 64, "gelu", True, FP), (5, 2048, 5632, 128, "silu", True, BF),
    (8, 4096, 14336, 32, "silu", False, FP), (17, 4160, 4160, 64, "relu", True, BF), (33, 2048, 8192, 128, "tanh", False, FP),
    (64, 4096, 14336, 64, "silu", False, BF), (64, 768, 2048, 32, "silu", True, FP)])
def test_mlp_at_serving_sizes(pkg, cuda_dev, M, K, N, group, act, bias, dt):
    g = _gen(cuda_dev, M + K)
    ws = [_w4(pkg, g, *s, group=group, symmetric=M == 33, dt=dt) for s in ((N, K), (N, K), (K, N))]
    bg, bu, bd = (_rnd(g, n, std=0.5, dt=dt) if bias else None for n in (N, N, K))
    x = _rnd(g, M, K, dt=dt)
    full = [ft.unpack(*w) for w in ws]
    y, limit = ft.mlp_rms(x, full[0], ws[0].scale, bg, full[1], ws[1].scale, bu, full[2], ws[2].scale, bd, dt, act)
    res = ft.cancelling_residual(y, dt)
    got = pkg.ops.kernels.decode_fwd_w4(x, ws[0], bg, ws[1], bu, ws[2], bd, act=act, residual=res)
    ft.check_rms(got, y, res, limit, dt, f"M={M} K={K} N={N} g{group}")


@pytest.mark.parametrize("T,E,k,K,N,group,dt", [
    (1, 64, 8, 2048, 768, 128, BF), (4, 16, 4, 2048, 1024, 64, FP), (6, 8, 2, 1024, 3584, 32, BF),
    (32, 32, 4, 2048, 896, 64, FP), (64, 24, 6, 1024, 704, 32, BF)])
def test_mixtures_at_serving_sizes(pkg, cuda_dev, T, E, k, K, N, group, dt):
    g = _gen(cuda_dev, T + E)
    ws = [_w4(pkg, g, E, *s, group=group, dt=dt) for s in ((N, K), (N, K), (K, N))]
    x = _rnd(g, T, K, dt=dt)
    ids = torch.stack([torch.randperm(E, generator=g, device=cuda_dev)[:k] for _ in range(T)]).to(torch.int32)
    wts = torch.rand((T, k), generator=g, device=cuda_dev) + 0.1
    full = [ft.unpack(*w) for w in ws]
    y, limit = ft.moe_rms(x, ids, wts, full[0], ws[0].scale, full[1], ws[1].scale, full[2], ws[2].scale, dt)
    res = ft.cancelling_residual(y, dt)
    got = pkg.ops.kernels.moe_decode_fwd_w4(x, ids, wts, *ws, residual=res)
    ft.check_rms(got, y, res, limit, dt, f"T={T} E={E} k={k} g{group}")
