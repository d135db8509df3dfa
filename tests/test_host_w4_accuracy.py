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


def _restated_mlp(x, wg, wu, wd, act, dt, group, terms):
    """decode_fwd_w4 with sums in 64 bits and activations of so many terms."""
    a = ft.as_terms(x, group, terms)
    h = (ft._ACTS[act](a @ wg.t()) * (a @ wu.t())).to(dt).double()
    return ft.as_terms(h, group, terms) @ wd.t()


@pytest.mark.parametrize("M,dt,group", [(3, BF, 128), (17, FP, 32), (64, BF, 64), (9, FP, 128)])
def test_mlp_limits_tell_three_terms_from_two(pkg, M, dt, group):
    g = torch.Generator().manual_seed(M)
    K, N = 512, 896
    (qg, wg), (qu, wu), (qd, wd) = (_w4(pkg, g, *s, group, dt) for s in ((N, K), (N, K), (K, N)))
    x = torch.randn((M, K), generator=g).to(dt).double()
    y, limit = ft.mlp_rms(x, wg, qg.scale, None, wu, qu.scale, None, wd, qd.scale, None, dt)
    res = ft.cancelling_residual(y, dt)
    ft.check_rms((_restated_mlp(x, wg, wu, wd, "silu", dt, group, 3) + res.double()).to(dt), y, res, limit, dt, "three")
    with pytest.raises(AssertionError, match="root-mean-square"):
        ft.check_rms((_restated_mlp(x, wg, wu, wd, "silu", dt, group, 2) + res.double()).to(dt), y, res, limit, dt, "two")


@pytest.mark.parametrize("T,dt,group", [(4, BF, 64), (20, FP, 64)])
def test_moe_limits_tell_three_terms_from_two(pkg, T, dt, group):
    g = torch.Generator().manual_seed(T)
    E, k, K, N = 6, 2, 256, 320
    packed = [pkg.ops.kernels.quantize_weight_int4((torch.randn((E, r, c), generator=g) * c ** -0.5).to(dt), group)
              for r, c in ((N, K), (N, K), (K, N))]
    wg, wu, wd = (ft.unpack(*q) for q in packed)
    x = torch.randn((T, K), generator=g).to(dt).double()
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    wts = torch.rand((T, k), generator=g) + 0.1
    y, limit = ft.moe_rms(x, ids, wts, wg, packed[0].scale, wu, packed[1].scale, wd, packed[2].scale, dt)
    res = ft.cancelling_residual(y, dt)
    for terms in (3, 2):
        top = wts.double().amax(1, keepdim=True)
        hs = torch.zeros((T, E, N), dtype=torch.float64)
        a = ft.as_terms(x, group, terms)
        for t in range(T):
            for j in range(k):
                e = int(ids[t, j])
                h = torch.nn.functional.silu(a[t] @ wg[e].t()) * (a[t] @ wu[e].t())
                hs[t, e] = (h * wts[t, j].double() / top[t]).to(dt).double()
        largest = None if T <= 4 else hs.abs().amax((1, 2), keepdim=True).flatten(1)
        got = top * ft.as_terms(hs.flatten(1), group, terms, largest) @ wd.transpose(0, 1).flatten(1).t()
        got = (got + res.double()).to(dt)
        if terms == 3:
            ft.check_rms(got, y, res, limit, dt, "three")
        else:
            with pytest.raises(AssertionError, match="root-mean-square"):
                ft.check_rms(got, y, res, limit, dt, "two")
