"""quantize_weight_int4 over the types' ranges and on views."""
import pytest
import torch

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dt,size", [(BF, 1e-9), (BF, 1e-30), (BF, 1e30), (FP, 1e-4), (FP, 1e3)])
def test_small_and_large_matrices_keep_their_values(pkg, dt, size, symmetric):
    """Half a step of a grid of 16 over the range, and what the rounding of scale and zero point moves its ends by."""
    K_ = pkg.ops.kernels
    w = (torch.randn((6, 128), generator=torch.Generator().manual_seed(1)).double() * size).to(dt)
    q = K_.quantize_weight_int4(w, 64, symmetric)
    step = q.scale.double().t().repeat_interleave(64, -1)
    off = (K_.dequantize_weight_int4(q).double() - w.double()).abs()
    # fp16's scale of 1e-4 / 4 has its last bit at 2^-24: half of it, sixteen times, on top
    assert (off <= step * (1 + 8 * torch.finfo(dt).eps) + (16 * 2.0 ** -25 if dt is FP else 0)).all()
    assert (off.pow(2).mean().sqrt() < w.double().pow(2).mean().sqrt() / 4)


@pytest.mark.parametrize("view", [lambda w: w.t().contiguous().t(), lambda w: w.repeat_interleave(2, 1)[:, ::2],
                                  lambda w: torch.cat([w, w], 1)[:, :w.shape[1]]])
def test_views_give_what_copies_give(pkg, view):
    K_ = pkg.ops.kernels
    w = torch.randn((40, 96), generator=torch.Generator().manual_seed(2)).to(BF)
    for a, b in zip(K_.quantize_weight_int4(view(w), 32), K_.quantize_weight_int4(w, 32)):
        assert a.is_contiguous() and torch.equal(a, b)
