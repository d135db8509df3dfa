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
