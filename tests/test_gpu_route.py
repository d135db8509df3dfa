"""The router on the inputs where a choice or a weight can go wrong: bad logits at every place of a lane's experts."""
import pytest
import torch

from oracle import few_token as ft

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rnd(g, *shape, std=1.0, dt=BF):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dt)


@pytest.mark.parametrize("E", [9, 40, 64, 300, 512])
@pytest.mark.parametrize("renormalize", [True, False])
def test_one_nan_logit_makes_every_weight_nan(pkg, cuda_dev, E, renormalize):
    """The softmax over all experts is NaN wherever in the list the NaN stands: first, middle and last of a lane's experts
    (lane l has l, l + 32, ...). The ids stay those of the numbers, with the NaN behind them."""
    g = _gen(cuda_dev, E)
    x, w = _rnd(g, 3, 64), _rnd(g, E, 64)
    k = min(E, 8)
    for bad in sorted({0, 8, E // 2, E - 1}):
        v = w.clone()
        v[bad, 5] = float("nan")
        ids, wts = pkg.ops.kernels.moe_route(x, v, k, renormalize=renormalize)
        assert torch.isnan(wts).all(), (bad, wts)
        logits = x.double() @ w.double().t()
        logits[:, bad] = -float("inf")
        assert torch.equal(ids.long(), torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]), bad


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("big", [100.0, 1000.0, 30000.0])
def test_large_channels_that_cancel(pkg, cuda_dev, dt, big):
    """Products of two channel pairs that are thousands of times a logit and cancel exactly, with others between them: the choice
    and the weights are those of the exact sums (64 bits: off by K 2^-53 of the products' magnitudes, below 2^-26 here)."""
    g = _gen(cuda_dev, int(big))
    for T, E, K, k in ((64, 64, 2048, 8), (3, 300, 1000, 32), (17, 7, 4096, 7)):
        x, w = _rnd(g, T, K, dt=dt), _rnd(g, E, K, std=K ** -0.5, dt=dt)
        x[:, 10], x[:, 11], x[:, 300], x[:, 301] = big, -big, big, -big
        w[:, 10:12], w[:, 300:302] = 1.0, 3.0
        ids, wts = pkg.ops.kernels.moe_route(x, w, k)
        want_ids, want = ft.route(x, w, k, True)
        assert torch.equal(ids, want_ids)
        # exp of a difference of logits, |d| <= ~20 in 32 bits, and a sum of E terms
        assert ((wts.double() - want).abs() <= want * 2.0 ** -17).all()


@pytest.mark.parametrize("dt", [BF, FP])
def test_every_magnitude_of_the_type(pkg, cuda_dev, dt):
    """Subnormals, the smallest and the largest numbers on both sides: logits as in 64 bits (one column of x is not zero)."""
    f = torch.finfo(dt)
    tiny = f.smallest_normal * f.eps
    scale = torch.tensor([tiny, 3 * tiny, f.smallest_normal, 1.0, f.max], dtype=torch.float64)
    w = torch.zeros(40, 64, dtype=dt)
    for i in range(40):
        w[i, i % 5] = (1 + (i // 5) / 8 * (1 if i % 5 > 2 else 0)) * scale[i % 5] / (2 if i % 5 == 4 else 1)
    for j in range(5):
        for v in (1.0, -1.0, tiny, f.max):
            x = torch.zeros(1, 64, dtype=dt)
            x[0, j] = v
            ids, wts = pkg.ops.kernels.moe_route(x.to(cuda_dev), w.to(cuda_dev), 32, renormalize=False)
            want_ids, want = ft.route(x, w, 32, False)
            assert torch.equal(ids.cpu(), want_ids), (j, v)
            assert ((wts.cpu().double() - want).abs() <= want * 2.0 ** -17 + 2.0 ** -126).all(), (j, v)


def test_infinite_router_weights(pkg, cuda_dev):
    """An infinite weight makes its expert the first or the last choice by the sign of x; its neighbours' logits stay."""
    g = _gen(cuda_dev, 1)
    for E in (12, 64, 200):
        x, w = _rnd(g, 6, 128), _rnd(g, E, 128)
        w[E // 2, 9] = float("inf")
        w[1, 100] = -float("inf")
        ids, wts = pkg.ops.kernels.moe_route(x, w, 10)
        logits = x.double() @ w.double().t()
        assert not torch.isnan(logits).any()
        assert torch.equal(ids.long(), torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :10])
        up = torch.isposinf(logits).any(1)
        assert torch.isnan(wts[up]).all()             # inf - inf, as in the formula
        _, want = ft.route(x[~up], w, 10, True)
        assert ((wts[~up].double() - want).abs() <= want * 2.0 ** -17).all()


@pytest.mark.parametrize("E,k", [(20, 3), (33, 6), (128, 8), (300, 32)])
def test_many_tokens(pkg, cuda_dev, E, k):
    """Enough tokens for two a cluster, an odd number of them: every token as in a call of its own, padding rows (zeros) and
    bad ones among them, and as in 64 bits."""
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, E)
    T = 2501
    for dt in (BF, FP):
        x, w = _rnd(g, T, 264, dt=dt), _rnd(g, E, 264, std=0.1, dt=dt)
        x[7], x[8, 3], x[T - 1], x[40, 0] = 0, float("nan"), 0, float("inf")
        ids, wts = K_.moe_route(x, w, k)
        ok = [t for t in range(T) if t not in (8, 40)]
        want_ids, want = ft.route(x[ok], w, k, True)
        assert torch.equal(ids[ok], want_ids)
        assert ((wts[ok].double() - want).abs() <= want * 2.0 ** -17).all()
        assert torch.isnan(wts[8]).all() and sorted(set(ids[8].tolist())) == sorted(ids[8].tolist())
        for t in (0, 7, 8, 40, 41, T - 1):
            one_ids, one = K_.moe_route(x[t:t + 1], w, k)
            assert torch.equal(one_ids, ids[t:t + 1])
            assert torch.allclose(one, wts[t:t + 1], rtol=2.0 ** -17, atol=0, equal_nan=True)
