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


@pytest.mark.parametrize("group", [32, 64, 128])
def test_group_size_of_a_weight_and_what_the_decode_path_takes(pkg, group):
    K_ = pkg.ops.kernels
    w = K_.quantize_weight_int4(torch.zeros(2, 40, 256, dtype=BF), group)
    assert w.group == group and K_.Int4Weight(*(t[0] for t in w)).group == group
    assert K_.decode_w4_supported(1, 256, 384, group) and K_.decode_w4_supported(64, 256, 384, group)
    for M, K, N, G in ((0, 256, 256, group), (65, 256, 256, group), (1, 256 + 16, 256, group), (1, 256, 16, group),
                       (1, 256, 256, 48)):
        assert not K_.decode_w4_supported(M, K, N, G)
