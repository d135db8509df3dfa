"""Hidden values beyond fp16 between the halves of a 4-bit MLP: stated to make their token's outputs NaN, and no other's."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FP = torch.float16


@pytest.mark.parametrize("M", [2, 4, 6, 40])
def test_overflowing_hidden_values_stay_in_their_token(pkg, cuda_dev, M):
    K_ = pkg.ops.kernels
    g = torch.Generator(device=cuda_dev).manual_seed(M)
    rnd = lambda *s: torch.randn(s, generator=g, device=cuda_dev)
    K, N, E = 256, 384, 4
    ws = [(rnd(E, *s) * s[1] ** -0.5).to(FP) for s in ((N, K), (N, K), (K, N))]
    q = [K_.quantize_weight_int4(w, 64) for w in ws]
    one = [K_.Int4Weight(*(t[0].contiguous() for t in w)) for w in q]
    x = rnd(M, K).to(FP)
    big = x.clone()
    big[1] *= 1000          # gate and up values around 1000: products around 1e6
    ids = (torch.arange(2 * M, device=cuda_dev, dtype=torch.int32) % E).view(M, 2)
    wts = torch.full((M, 2), 0.5, device=cuda_dev)
    rest = [m for m in range(M) if m != 1]
    for call in (lambda v: K_.decode_fwd_w4(v, one[0], None, one[1], None, one[2], None),
                 lambda v: K_.moe_decode_fwd_w4(v, ids, wts, *q)):
        a, b = call(x), call(big)
        assert torch.isfinite(a).all() and torch.equal(a[rest], b[rest])
        assert torch.isnan(b[1]).all()
