"""Products with 4-bit weights, the gated MLP on them, the router and the mixture-of-experts layers against their 64-bit
restatement (oracle/few_token.py), whose bounds count the roundings the kernels are allowed."""
import pytest
import torch

from oracle import few_token as ft

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rnd(g, *shape, std=1.0, dt=BF):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dt)


def _w4(pkg, g, *shape, group, symmetric, dt):
    return pkg.ops.kernels.quantize_weight_int4(_rnd(g, *shape, std=shape[-1] ** -0.5, dt=dt), group, symmetric)


def _unpack(w):
    return ft.unpack(*w)


@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("rows,cols,group", [(256, 256, 128), (129, 384, 64), (1, 32, 32), (1000, 1184, 32),
                                             (300, 128, 128), (4096, 2048, 128)])
def test_linear_w4(pkg, cuda_dev, M, rows, cols, group):
    dt = BF if (M + rows) % 2 else FP
    g = _gen(cuda_dev, M * 7 + rows)
    w = _w4(pkg, g, rows, cols, group=group, symmetric=M % 3 == 0, dt=dt)
    x = _rnd(g, M, cols, dt=dt)
    bias = _rnd(g, rows, dt=dt) if M % 2 else None
    res = _rnd(g, M, rows, dt=dt) if M % 4 else None
    y = pkg.ops.kernels.linear_w4(x, w, bias=bias, residual=res)
    ft.check(y, *ft.linear(x, _unpack(w), bias, res, dt, group), f"linear_w4 M={M} {rows}x{cols} g{group}")


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 16, 17, 64])
@pytest.mark.parametrize("dt,group", [(BF, 128), (FP, 32)])
def test_linear_w4_many_units_per_block(pkg, cuda_dev, M, dt, group):
    """Every ring of the stream kernel turns several times (about 14 units of 65,536 weights per block)."""
    g = _gen(cuda_dev, M)
    w = _w4(pkg, g, 16384, 8192, group=group, symmetric=False, dt=dt)
    x = _rnd(g, M, 8192, dt=dt)
    y = pkg.ops.kernels.linear_w4(x, w)
    ft.check(y, *ft.linear(x, _unpack(w), None, None, dt, group), f"linear_w4 M={M} g{group}")


def test_linear_w4_every_nibble_and_zero(pkg, cuda_dev):
    """All 16 values against all 16 zeros, one column at a time: exact."""
    K_ = pkg.ops.kernels
    for dt in (BF, FP):
        rows, cols = 256, 64
        q = (torch.arange(rows, device=cuda_dev) % 16)[:, None].expand(rows, cols).to(torch.int32)
        shifts = torch.tensor(K_.INT4_SHIFTS, dtype=torch.int32, device=cuda_dev)
        words = (q.unflatten(-1, (-1, 8)) << shifts).sum(-1).to(torch.int32)
        zero = (torch.arange(rows, device=cuda_dev) // 16).to(torch.uint8).expand(2, rows).contiguous()
        w = K_.Int4Weight(words.view(torch.uint8).contiguous(), torch.ones((2, rows), dtype=dt, device=cuda_dev), zero)
        x = torch.eye(cols, dtype=dt, device=cuda_dev)
        y = K_.linear_w4(x, w)
        want = (torch.arange(rows, device=cuda_dev) % 16 - torch.arange(rows, device=cuda_dev) // 16).to(dt)
        assert torch.equal(y, want.expand(cols, rows))


@pytest.mark.parametrize("M,K,N,group,act,bias", [(1, 256, 384, 128, "silu", False), (3, 512, 896, 128, "gelu", True),
                                                  (16, 320, 576, 64, "relu", True), (20, 288, 416, 32, "tanh", True),
                                                  (33, 1024, 640, 64, "leaky_relu", False),
                                                  (64, 768, 2048, 128, "silu", True), (5, 128, 128, 128, "no_act", False),
                                                  (48, 512, 512, 32, "sigmoid", True)])
@pytest.mark.parametrize("dt", [BF, FP])
def test_decode_fwd_w4(pkg, cuda_dev, M, K, N, group, act, bias, dt):
    g = _gen(cuda_dev, M + K + N)
    wg, wu = (_w4(pkg, g, N, K, group=group, symmetric=M % 2 == 0, dt=dt) for _ in range(2))
    wd = _w4(pkg, g, K, N, group=group, symmetric=M % 2 == 0, dt=dt)
    bg, bu, bd = (_rnd(g, n, dt=dt) if bias else None for n in (N, N, K))
    x = _rnd(g, M, K, dt=dt)
    res = _rnd(g, M, K, dt=dt) if M % 2 else None
    y = pkg.ops.kernels.decode_fwd_w4(x, wg, bg, wu, bu, wd, bd, act=act, residual=res)
    ft.check(y, *ft.mlp(x, _unpack(wg), bg, _unpack(wu), bu, _unpack(wd), bd, res, dt, act, group),
             f"decode_fwd_w4 M={M} K={K} N={N} g{group} {act}")


@pytest.mark.parametrize("M,K,E,k", [(1, 64, 4, 2), (5, 576, 18, 3), (64, 2048, 128, 8), (3, 256, 512, 32), (2, 8, 1, 1),
                                     (130, 1024, 33, 6), (7, 4096, 8, 8)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_moe_route(pkg, cuda_dev, M, K, E, k, renormalize):
    for dt in (BF, FP):
        g = _gen(cuda_dev, M + E)
        x, w = _rnd(g, M, K, dt=dt), _rnd(g, E, K, std=1.5 * K ** -0.5, dt=dt)
        ids, wts = pkg.ops.kernels.moe_route(x, w, k, renormalize=renormalize)
        want_ids, want = ft.route(x, w, k, renormalize)
        assert torch.equal(ids, want_ids)
        # exp of a difference of logits (|d| <= ~20, each logit within 2^-22 of its size) and a sum of E terms
        assert ((wts.double() - want).abs() <= want * 2.0 ** -17).all()


def _moe_inputs(g, T, E, k, K, N, dt):
    x = _rnd(g, T, K, dt=dt)
    ids = torch.stack([torch.randperm(E, generator=g, device=g.device)[:k] for _ in range(T)]).to(torch.int32)
    w = torch.rand((T, k), generator=g, device=g.device)
    return x, ids, w / w.sum(1, keepdim=True)


MOE_CASES = [(1, 8, 2, 256, 384), (5, 18, 3, 576, 320), (16, 4, 4, 128, 64), (17, 40, 6, 192, 128), (33, 3, 2, 320, 704),
             (64, 64, 6, 256, 192), (64, 2, 1, 1024, 512), (2, 512, 1, 64, 64), (9, 1, 1, 64, 192)]


@pytest.mark.parametrize("T,E,k,K,N", MOE_CASES)
@pytest.mark.parametrize("dt", [BF, FP])
def test_moe_decode_fwd(pkg, cuda_dev, T, E, k, K, N, dt):
    g = _gen(cuda_dev, T + E + K)
    x, ids, wts = _moe_inputs(g, T, E, k, K, N, dt)
    wg, wu, wd = (_rnd(g, E, *s, std=s[1] ** -0.5, dt=dt) for s in ((N, K), (N, K), (K, N)))
    res = _rnd(g, T, K, dt=dt) if T % 2 else None
    y = pkg.ops.kernels.moe_decode_fwd(x, ids, wts, wg, wu, wd, residual=res)
    ft.check(y, *ft.moe(x, ids, wts, wg.double(), wu.double(), wd.double(), res, dt), f"moe T={T} E={E} k={k}")


@pytest.mark.parametrize("T,E,k,K,N", [c for c in MOE_CASES])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_moe_decode_fwd_w4(pkg, cuda_dev, T, E, k, K, N, group):
    dt = BF if group == 64 else FP
    K, N = (-(-v // group) * group for v in (K, N))
    g = _gen(cuda_dev, T + E + K)
    x, ids, wts = _moe_inputs(g, T, E, k, K, N, dt)
    wg, wu = (_w4(pkg, g, E, N, K, group=group, symmetric=T % 2 == 0, dt=dt) for _ in range(2))
    wd = _w4(pkg, g, E, K, N, group=group, symmetric=T % 2 == 0, dt=dt)
    res = _rnd(g, T, K, dt=dt) if T % 2 else None
    y = pkg.ops.kernels.moe_decode_fwd_w4(x, ids, wts, wg, wu, wd, residual=res)
    ft.check(y, *ft.moe(x, ids, wts, _unpack(wg), _unpack(wu), _unpack(wd), res, dt, group=group),
             f"moe w4 T={T} E={E} k={k} g{group}")


@pytest.mark.parametrize("four_bit", [False, True])
def test_moe_padding_repeats_and_nothing_chosen(pkg, cuda_dev, four_bit):
    """ids of -1 (and past the end) are skipped, a repeated expert adds, a token with no expert keeps its residual, and a
    call in which no token chose anything returns the residual, or zero."""
    K_ = pkg.ops.kernels
    T, E, k, K, N, dt = 6, 5, 3, 256, 384, BF
    g = _gen(cuda_dev, 3)
    x, ids, wts = _moe_inputs(g, T, E, k, K, N, dt)
    ids[1] = -1
    ids[2, 1] = 999
    ids[3, 2] = ids[3, 0]
    wts[4] = 0.0
    x[1] = float("nan")   # a padded row's garbage stays in its row
    ws = [_rnd(g, E, *s, std=s[1] ** -0.5, dt=dt) for s in ((N, K), (N, K), (K, N))]
    if four_bit:
        packed = [K_.quantize_weight_int4(w, 128) for w in ws]
        full = [_unpack(w) for w in packed]
        fn = lambda i, r: K_.moe_decode_fwd_w4(x, i, wts, *packed, residual=r)
    else:
        full = [w.double() for w in ws]
        fn = lambda i, r: K_.moe_decode_fwd(x, i, wts, *ws, residual=r)
    res = _rnd(g, T, K, dt=dt)
    for r in (res, None):
        y = fn(ids, r)
        want, bound = ft.moe(torch.nan_to_num(x), ids, wts, *full, r, dt, group=128)
        ft.check(y, want, bound, "moe with padding")
        assert torch.equal(y[1], r[1] if r is not None else torch.zeros_like(y[1]))
        none = torch.full_like(ids, -1)
        y = fn(none, r)
        assert torch.equal(y, r if r is not None else torch.zeros_like(y))
