"""The few-token operators without a GPU: the 4-bit format, buffer sizes, what the C entries and the Python entries refuse,
and the modules' surface."""
import ctypes as C

import pytest
import torch

from oracle import few_token as ft

BF, FP = torch.bfloat16, torch.float16
A = 1 << 20          # an aligned address; every call below is refused before anything reads it
ARG, SHAPE, ALIGN, DTYPE, SCRATCH = -6, -1, -2, -3, -7


# ------------------------------------------------------------------ format --
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dt", [BF, FP])
def test_quantizer_and_format(pkg, group, symmetric, dt):
    K_ = pkg.ops.kernels
    g = torch.Generator().manual_seed(group)
    w = torch.randn((3, 5, 2 * group), generator=g).to(dt)
    q = K_.quantize_weight_int4(w, group, symmetric)
    assert q.w4.shape == (3, 5, group) and q.w4.dtype is torch.uint8
    assert q.scale.shape == (3, 2, 5) and q.scale.dtype is dt and q.scale.is_contiguous()
    assert (q.zero is None) == symmetric and (symmetric or q.zero.shape == (3, 2, 5))
    full = K_.dequantize_weight_int4(q).double()
    assert torch.equal(full, ft.unpack(*q))          # (q - zero) * scale is exact in float32: 4 + 11 bits
    # Off by half a step of the grid, and where the grid's end is clamped by what the rounding of the scale (half
    # an ulp of dt of up to 16 steps) and of the zero point (half a step) moved it
    step = q.scale.double().transpose(-1, -2).repeat_interleave(group, -1)
    eps = torch.finfo(dt).eps / 2
    assert ((full - w.double()).abs() <= step * (1.0 + 16 * eps)).all()


def test_quantizer_refuses(pkg):
    q = pkg.ops.kernels.quantize_weight_int4
    with pytest.raises(ValueError, match="group size"):
        q(torch.zeros(4, 96, dtype=BF), 48)
    with pytest.raises(ValueError, match="no multiple"):
        q(torch.zeros(4, 96, dtype=BF), 64)
    with pytest.raises(NotImplementedError):
        q(torch.zeros(4, 96), 32)


def test_zero_weights_and_wide_range_quantize(pkg):
    K_ = pkg.ops.kernels
    w = torch.zeros(2, 64, dtype=FP)
    assert torch.equal(K_.dequantize_weight_int4(K_.quantize_weight_int4(w, 32)), w.float())
    w[0, 3], w[1, 40] = 60000.0, -60000.0
    full = K_.dequantize_weight_int4(K_.quantize_weight_int4(w, 32))
    assert torch.isfinite(full).all() and (full - w.float()).abs().max() <= 60000.0 / 15


# ------------------------------------------------------------ buffer sizes --
def test_buffer_sizes(pkg):
    lib = pkg._lib.load()
    front = lib.gmlp_few_scratch_counters()
    assert front > 0 and front % 256 == 0
    for K, N, E in ((4096, 14336, 1), (64, 64, 512), (1, 1, 1), (8192, 131072, 128)):
        n = lib.gmlp_few_scratch_bytes(K, N, E)
        assert n >= front + 4 * (-(-N // 128) * E + -(-K // 128))
        assert lib.gmlp_few_scratch_bytes(K, 2 * N, E) >= n
    for bad in ((0, 64, 1), (64, 0, 1), (64, 64, 0), (64, 64, 513), (-1, 64, 1)):
        assert lib.gmlp_few_scratch_bytes(*bad) == 0
    # up to four tokens there is only the hidden state; more have their terms too (two a value in bf16, three in fp16)
    assert lib.gmlp_w4_work_bytes(4, 256, 512, 3, 128, 0) == 3 * 4 * 512 * 2
    for dt, terms in ((0, 2), (1, 3)):
        n = lib.gmlp_w4_work_bytes(64, 256, 512, 3, 32, dt)
        assert n >= 3 * 64 * 512 * (2 + terms)
    for bad in ((0, 64, 64, 1, 32, 0), (65, 64, 64, 1, 32, 0), (1, 0, 64, 1, 32, 0), (1, 64, -1, 1, 32, 0),
                (1, 64, 64, 0, 32, 0), (1, 64, 64, 1, 48, 0)):
        assert lib.gmlp_w4_work_bytes(*bad) == 0


# -------------------------------------------------------- C entries' refusals --
LINEAR = dict(M=4, rows=256, cols=256, group=128, dtype=0, x=A, ldx=256, w4=A, scale=A, zero=A, bias=None, residual=None,
              y=A, work=A, work_bytes=1 << 40, scratch=A, scratch_bytes=1 << 40, tuning=0, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(M=0), SHAPE), (dict(M=65), SHAPE), (dict(M=-3), SHAPE), (dict(rows=0), SHAPE), (dict(cols=0), SHAPE),
    (dict(rows=1 << 31), SHAPE), (dict(group=96), SHAPE), (dict(group=0), SHAPE), (dict(cols=192, ldx=192), SHAPE),
    (dict(dtype=2), DTYPE), (dict(dtype=9), DTYPE), (dict(x=None), ARG), (dict(y=None), ARG), (dict(work=None), ARG),
    (dict(scratch=None), ARG), (dict(w4=None), ARG), (dict(scale=None), ARG), (dict(x=A + 2), ALIGN),
    (dict(w4=A + 8), ALIGN), (dict(scale=A + 2), ALIGN), (dict(zero=A + 1), ALIGN), (dict(scratch=A + 4), ALIGN),
    (dict(ldx=248), ALIGN), (dict(ldx=260), ALIGN)])
def test_w4_linear_refuses(pkg, change, code):
    lib = pkg._lib.load()
    assert lib.gmlp_w4_linear(*{**LINEAR, **change}.values()) == code
    assert lib.gmlp_last_error()


def _problem(pkg, **kw):
    p = pkg._lib.Problem()
    p.M, p.K, p.N, p.dtype, p.dropout_p = 4, 256, 512, 0, 0.0
    p.N_global, p.act, p.tuning = 512, pkg.ops.kernels.act_code("silu"), 0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


MLP = dict(group=128, x=A, wg=A, sg=A, zg=A, bg=None, wu=A, su=A, zu=A, bu=None, wd=A, sd=A, zd=None, bd=None, residual=None,
           y=A, work=A, work_bytes=1 << 40, scratch=A, scratch_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("problem,change,code", [
    (dict(M=65), {}, SHAPE), (dict(M=0), {}, SHAPE), (dict(K=264), {}, SHAPE), (dict(N=576, N_global=576), {}, SHAPE),
    (dict(dtype=2), {}, DTYPE), (dict(dropout_p=0.5), {}, ARG), ({}, dict(group=16), SHAPE), ({}, dict(zu=None), ARG),
    ({}, dict(zg=None), ARG), ({}, dict(wd=None), ARG), ({}, dict(sd=A + 1), ALIGN), ({}, dict(wu=A + 4), ALIGN),
    ({}, dict(x=A + 8), ALIGN), ({}, dict(work=None), ARG)])
def test_decode_fwd_w4_refuses(pkg, problem, change, code):
    lib = pkg._lib.load()
    assert lib.gmlp_decode_fwd_w4(C.byref(_problem(pkg, **problem)), *{**MLP, **change}.values()) == code


MOE = dict(experts=8, top_k=2, x=A, ids=A, weights=A, wg=A, wu=A, wd=A, residual=None, h=A, y=A, scratch=A,
           scratch_bytes=1 << 40, stream=None)
MOE_W4 = dict(group=128, experts=8, top_k=2, x=A, ids=A, weights=A, wg=A, sg=A, zg=A, wu=A, su=A, zu=A, wd=A, sd=A,
              zd=None, residual=None, y=A, work=A, work_bytes=1 << 40, scratch=A, scratch_bytes=1 << 40, stream=None)
MOE_BAD = [(dict(M=65), {}, SHAPE), (dict(dropout_p=0.1), {}, ARG), (dict(dtype=2), {}, DTYPE), ({}, dict(experts=0), SHAPE),
           ({}, dict(experts=513), SHAPE), ({}, dict(top_k=0), SHAPE), ({}, dict(top_k=9), SHAPE),
           ({}, dict(experts=64, top_k=33), SHAPE), ({}, dict(ids=None), ARG), ({}, dict(weights=None), ARG),
           ({}, dict(ids=A + 2), ALIGN), ({}, dict(x=A + 4), ALIGN), ({}, dict(y=None), ARG),
           (dict(N=1 << 30, N_global=1 << 30), {}, SHAPE)]


@pytest.mark.parametrize("problem,change,code", MOE_BAD + [(dict(K=288), {}, SHAPE), ({}, dict(wu=None), ARG),
                                                           ({}, dict(h=None), ARG)])
def test_moe_decode_fwd_refuses(pkg, problem, change, code):
    lib = pkg._lib.load()
    assert lib.gmlp_moe_decode_fwd(C.byref(_problem(pkg, **problem)), *{**MOE, **change}.values()) == code


@pytest.mark.parametrize("problem,change,code", MOE_BAD + [(dict(K=320), {}, SHAPE), ({}, dict(zu=None), ARG),
                                                           ({}, dict(scratch=None), ARG)])
def test_moe_decode_fwd_w4_refuses(pkg, problem, change, code):
    lib = pkg._lib.load()
    assert lib.gmlp_moe_decode_fwd_w4(C.byref(_problem(pkg, **problem)), *{**MOE_W4, **change}.values()) == code


ROUTE = dict(M=4, K=256, experts=8, top_k=2, renormalize=1, dtype=0, x=A, ldx=256, w=A, ids=A, weights=A, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(M=0), SHAPE), (dict(K=0), SHAPE), (dict(K=252, ldx=256), SHAPE), (dict(experts=0), SHAPE),
    (dict(experts=513), SHAPE), (dict(top_k=9), SHAPE), (dict(top_k=0), SHAPE), (dict(dtype=2), DTYPE),
    (dict(x=None), ARG), (dict(ids=None), ARG), (dict(weights=None), ARG), (dict(x=A + 2), ALIGN), (dict(w=A + 2), ALIGN),
    (dict(ldx=248), ALIGN), (dict(ldx=257), ALIGN), (dict(ids=A + 1), ALIGN), (dict(M=1 << 24), SHAPE)])
def test_moe_route_refuses(pkg, change, code):
    lib = pkg._lib.load()
    assert lib.gmlp_moe_route(*{**ROUTE, **change}.values()) == code


def test_capture_id_refuses_null(pkg):
    assert pkg._lib.load().gmlp_capture_id(None, None) == ARG


# ---------------------------------------------------- Python entries' refusals --
def test_cpu_tensors_are_refused(pkg):
    """No CPU path: the tensors' device is the first thing that is looked at."""
    K_, err = pkg.ops.kernels, pkg._lib.GmlpError
    x = torch.zeros(2, 128, dtype=BF)
    w = K_.quantize_weight_int4(torch.zeros(128, 128, dtype=BF), 128)
    e = K_.Int4Weight(*(t[None] for t in w))
    ids, wts = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1)
    full = torch.zeros(1, 128, 128, dtype=BF)
    for call in (lambda: K_.linear_w4(x, w), lambda: K_.decode_fwd_w4(x, w, None, w, None, w, None),
                 lambda: K_.moe_route(x, full[0], 1), lambda: K_.moe_decode_fwd(x, ids, wts, full, full, full),
                 lambda: K_.moe_decode_fwd_w4(x, ids, wts, e, e, e)):
        with pytest.raises(err, match="no CPU path"):
            call()


# ------------------------------------------------------------------ modules --
def test_module_quantize_arguments(pkg):
    m = pkg.FusedGatedMLP(192, 384, bias=False).to(BF)
    with pytest.raises(NotImplementedError, match="4 and 8"):
        m.quantize_decode_weights(bits=3)
    with pytest.raises(ValueError, match="group size"):
        m.quantize_decode_weights(bits=4, group_size=128)
    with pytest.raises(ValueError, match="multiples of 128"):
        m.quantize_decode_weights()
    m.quantize_decode_weights(bits=4, group_size=64)
    assert m._w4[0].w4.shape == (384, 96) and m._w4[2].scale.shape == (6, 192) and m._fp8 is None
    with pytest.raises(NotImplementedError, match="input norm"):
        m.attach_input_norm(torch.ones(192))
    m.quantize_decode_weights(False)
    assert m._w4 is None
    m.attach_input_norm(torch.ones(192))
    with pytest.raises(NotImplementedError, match="input norm"):
        m.quantize_decode_weights(bits=4, group_size=64)


def test_moe_module_surface(pkg):
    m = pkg.FusedMoEGatedMLP(128, 192, 6, 2)
    assert [n for n, _ in m.named_parameters()] == ["gate_proj", "up_proj", "down_proj", "router.weight"]
    assert m.gate_proj.shape == m.up_proj.shape == (6, 192, 128) and m.down_proj.shape == (6, 128, 192)
    assert m.router.weight.shape == (6, 128)
    twin = pkg.FusedMoEGatedMLP(128, 192, 6, 2)
    twin.load_state_dict(m.state_dict())
    assert torch.equal(twin.down_proj, m.down_proj)
    m = m.to(BF)
    m.quantize_decode_weights(group_size=64)
    assert m._w4[0].w4.shape == (6, 192, 64) and m._w4[2].zero.shape == (6, 3, 128)
    m.quantize_decode_weights(False)
    assert m._w4 is None


def test_moe_module_refuses(pkg):
    mod = pkg.FusedMoEGatedMLP
    for args in ((128, 192, 0, 1), (128, 192, 513, 1), (128, 192, 4, 0), (128, 192, 4, 5), (128, 192, 64, 33),
                 (100, 192, 4, 2), (128, 200, 4, 2), (0, 64, 4, 2)):
        with pytest.raises(ValueError):
            mod(*args)
    with pytest.raises(NotImplementedError):
        mod(128, 192, 4, 2, hidden_act="mish")
    m = mod(128, 192, 4, 2).to(BF)
    x = torch.zeros(3, 128, dtype=BF)
    with pytest.raises(NotImplementedError, match="no backward"):
        m(x)
    with torch.no_grad():
        with pytest.raises(pkg._lib.GmlpError, match="no CPU path"):
            m(x)
        with pytest.raises(ValueError, match="residual shape"):
            m(x, residual=x[:2])
    with pytest.raises(NotImplementedError, match="8-bit"):
        m.quantize_decode_weights(bits=8)
    with pytest.raises(ValueError, match="group size"):
        m.quantize_decode_weights(group_size=128)
