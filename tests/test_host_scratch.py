"""Scratch buffers that callers bring: refused before anything is launched where a kernel would write to memory that is not
its device's, or not the buffer's."""
import pytest
import torch


def test_scratch_elsewhere_or_in_pieces_is_refused(pkg):
    K_ = pkg.ops.kernels
    dev = torch.device("cuda", 0)
    for bad in (torch.zeros(1 << 16, dtype=torch.uint8), torch.zeros(1 << 16, dtype=torch.uint8, device="meta"),
                torch.zeros(1 << 17, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="scratch must be"):
            K_._few_buffers(bad, 256, 256, 1, 1024, dev, 0)
    with pytest.raises(ValueError, match="scratch must be"):
        K_._check_scratch(torch.zeros(64, dtype=torch.int32)[::2], torch.device("cpu"))
    K_._check_scratch(torch.zeros(64, dtype=torch.int32), torch.device("cpu"))


@pytest.mark.gpu
def test_every_call_with_a_scratch_refuses_another_devices(pkg, cuda_dev):
    K_, BF = pkg.ops.kernels, torch.bfloat16
    x, w = torch.zeros(2, 128, dtype=BF, device=cuda_dev), torch.zeros(128, 128, dtype=BF, device=cuda_dev)
    q = K_.quantize_weight_int4(w, 128)
    e = K_.Int4Weight(*(t[None] for t in q))
    w8, s8 = K_.quantize_weight_rows_e4m3(w)
    ids, wts = torch.zeros(2, 1, dtype=torch.int32, device=cuda_dev), torch.ones(2, 1, device=cuda_dev)
    whole = torch.zeros(1 << 26, dtype=torch.uint8, device=cuda_dev)
    for bad in (torch.zeros(1 << 26, dtype=torch.uint8), whole[::2]):
        for call in (lambda: K_.linear_w4(x, q, scratch=bad),
                     lambda: K_.decode_fwd_w4(x, q, None, q, None, q, None, scratch=bad),
                     lambda: K_.moe_decode_fwd(x, ids, wts, w[None], w[None], w[None], scratch=bad),
                     lambda: K_.moe_decode_fwd_w4(x, ids, wts, e, e, e, scratch=bad),
                     lambda: K_.decode_fwd(x, w, None, w, None, w, None, scratch=bad),
                     lambda: K_.decode_fwd_fp8(x, w8, s8, None, w8, s8, None, w8, s8, None, scratch=bad)):
            with pytest.raises(ValueError, match="scratch must be"):
                call()
    assert not whole.any()
