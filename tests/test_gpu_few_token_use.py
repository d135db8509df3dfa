"""The few-token operators as they are used: through the modules and one after the other, captured and replayed, on
several streams, with padded and pitched inputs, at the ends of their ranges, and on bad numbers."""
import pytest
import torch

from oracle import few_token as ft

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _rnd(g, *shape, std=1.0, dt=BF):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dt)


def _w4(pkg, g, *shape, group=128, symmetric=False, dt=BF):
    return pkg.ops.kernels.quantize_weight_int4(_rnd(g, *shape, std=shape[-1] ** -0.5, dt=dt), group, symmetric)


def _choices(g, T, E, k):
    ids = torch.stack([torch.randperm(E, generator=g, device=g.device)[:k] for _ in range(T)]).to(torch.int32)
    w = torch.rand((T, k), generator=g, device=g.device) + 0.1
    return ids, w / w.sum(1, keepdim=True)


def _calls(pkg, dev, M, dt=BF, seed=0):
    """name -> closure: one call of every operator for M tokens, each with inputs of its own."""
    K_ = pkg.ops.kernels
    g = _gen(dev, seed + M)
    K, N, E, k = 512, 640, 12, 3
    x = _rnd(g, M, K, dt=dt)
    wl = _w4(pkg, g, 1000, K, dt=dt)
    dense = [_w4(pkg, g, *s, dt=dt) for s in ((N, K), (N, K), (K, N))]
    experts = [_rnd(g, E, *s, std=s[1] ** -0.5, dt=dt) for s in ((N, K), (N, K), (K, N))]
    experts4 = [K_.quantize_weight_int4(w, 128) for w in experts]
    router = _rnd(g, E, K, std=K ** -0.5, dt=dt)
    ids, wts = _choices(g, M, E, k)
    return {
        "linear_w4": lambda **kw: K_.linear_w4(x, wl, **kw),
        "decode_fwd_w4": lambda **kw: K_.decode_fwd_w4(x, dense[0], None, dense[1], None, dense[2], None, **kw),
        "moe_route": lambda **kw: torch.cat([t.float() for t in K_.moe_route(x, router, k)]),
        "moe_decode_fwd": lambda **kw: K_.moe_decode_fwd(x, ids, wts, *experts, **kw),
        "moe_decode_fwd_w4": lambda **kw: K_.moe_decode_fwd_w4(x, ids, wts, *experts4, **kw),
    }


@pytest.mark.parametrize("M", [1, 4, 5, 16, 33, 64])
def test_same_bits_every_time(pkg, cuda_dev, M):
    for name, call in _calls(pkg, cuda_dev, M, BF if M % 2 else FP).items():
        first = call()
        for _ in range(5):
            assert torch.equal(call(), first), name


# -------------------------------------------------------- graphs and streams --
@pytest.mark.parametrize("M", [1, 6, 64])
def test_two_graphs_and_eager_calls_together(pkg, cuda_dev, M):
    """Two graphs of every operator, replayed at once on two streams while eager calls run on a third."""
    calls = _calls(pkg, cuda_dev, M)
    want = {n: c() for n, c in calls.items()}
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = {n: c() for n, c in calls.items()}
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(10):
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        for n, c in calls.items():
            assert torch.equal(c(), want[n]), n
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        for n, v in out.items():
            assert torch.equal(v, want[n]), n


def test_one_graph_captured_over_two_streams(pkg, cuda_dev):
    """A capture that forks: the branches may run at once and do not share counters."""
    calls = _calls(pkg, cuda_dev, 9)
    want = {n: c() for n, c in calls.items()}
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = {n: c() for n, c in calls.items()}
        a = {n: c() for n, c in calls.items()}
        main.wait_stream(side)
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(a[n], want[n]) and torch.equal(b[n], want[n]), n


def test_two_streams_at_once(pkg, cuda_dev):
    sets = [_calls(pkg, cuda_dev, M, seed=7 * M) for M in (3, 20)]
    want = [{n: c() for n, c in s.items()} for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for s, calls, out in zip(streams, sets, got):
            with torch.cuda.stream(s):
                out.append({n: c() for n, c in calls.items()})
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        for o in out:
            for n in w:
                assert torch.equal(o[n], w[n]), n


def test_own_scratch_serves_calls_of_other_shapes(pkg, cuda_dev):
    K_ = pkg.ops.kernels
    scratch = K_.few_scratch(4096, 4096, 64, cuda_dev)
    for M in (64, 1, 17):
        for name, call in _calls(pkg, cuda_dev, M).items():
            if name != "moe_route":
                assert torch.equal(call(scratch=scratch), call()), name
    small = torch.zeros(1024, dtype=torch.uint8, device=cuda_dev)
    with pytest.raises(pkg._lib.GmlpError, match="scratch holds"):
        _calls(pkg, cuda_dev, 1)["linear_w4"](scratch=small)


@pytest.mark.parametrize("M", [2, 40])
def test_weights_written_by_the_kernel_before(pkg, cuda_dev, M):
    """ordinary_launch: a copy that takes a while writes the weights that the call reads."""
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    a, b = (_w4(pkg, g, 2048, 2048) for _ in range(2))
    x = _rnd(g, M, 2048)
    want = K_.linear_w4(x, b), K_.decode_fwd_w4(x, b, None, b, None, b, None)
    buf = K_.Int4Weight(*(t.clone() for t in a))
    filler = torch.empty(1 << 28, dtype=torch.uint8, device=cuda_dev)
    for i, call in enumerate((lambda: K_.linear_w4(x, buf, ordinary_launch=True),
                              lambda: K_.decode_fwd_w4(x, buf, None, buf, None, buf, None, ordinary_launch=True))):
        for t, s in zip(buf, a):
            t.copy_(s)
        filler.zero_()
        for t, s in zip(buf, b):
            t.copy_(s)
        assert torch.equal(call(), want[i])


# ------------------------------------------------------------ odd inputs --
@pytest.mark.parametrize("M", [1, 3, 7, 64])
def test_pitched_and_misaligned_inputs(pkg, cuda_dev, M):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    K, N, E, k = 320, 448, 6, 2
    wide = _rnd(g, M, K + 72)
    x = wide[:, 8:8 + K].contiguous()
    pitched = wide[:, 8:8 + K]
    odd = torch.empty(M * K + 1, dtype=BF, device=cuda_dev)[1:].view(M, K).copy_(x)
    turned = x.t().contiguous().t()
    wl = _w4(pkg, g, 333, K, group=64)
    dense = [_w4(pkg, g, *s, group=64) for s in ((N, K), (N, K), (K, N))]
    experts = [_rnd(g, E, *s, std=s[1] ** -0.5) for s in ((N, K), (N, K), (K, N))]
    router = _rnd(g, E, K, std=K ** -0.5)
    ids, wts = _choices(g, M, E, k)
    res = _rnd(g, K, M).t()
    for call in (lambda v: K_.linear_w4(v, wl), lambda v: K_.decode_fwd_w4(v, dense[0], None, dense[1], None, dense[2], None,
                                                                            residual=res),
                 lambda v: K_.moe_route(v, router, k)[1],
                 lambda v: K_.moe_decode_fwd(v, ids, wts, *experts, residual=res)):
        want = call(x)
        for v in (pitched, odd, turned):
            assert torch.equal(call(v), want)
    # the routing table as a transposed view, the experts' weights as one
    assert torch.equal(K_.moe_decode_fwd(x, ids.t().contiguous().t(), wts.t().contiguous().t(), *experts),
                       K_.moe_decode_fwd(x, ids, wts, *(w.transpose(1, 2).contiguous().transpose(1, 2) for w in experts)))


@pytest.mark.parametrize("M", [1, 4, 5, 12, 64])
@pytest.mark.parametrize("rows,cols,group", [(1001, 352, 32), (127, 192, 64), (2, 384, 128), (515, 96, 32), (24, 4160, 64)])
def test_linear_w4_rows_that_are_not_aligned(pkg, cuda_dev, M, rows, cols, group):
    """Scales and zeros copied word by word, from rows that start up to three bytes into a word."""
    g = _gen(cuda_dev, M + rows)
    for dt in (BF, FP):
        w = _w4(pkg, g, rows, cols, group=group, dt=dt)
        x = _rnd(g, M, cols, dt=dt)
        y = pkg.ops.kernels.linear_w4(x, w)
        ft.check(y, *ft.linear(x, ft.unpack(*w), None, None, dt, group), f"M={M} {rows}x{cols} g{group}")


def test_no_tokens(pkg, cuda_dev):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, 1)
    x = torch.empty(0, 128, dtype=BF, device=cuda_dev)
    w = _w4(pkg, g, 128, 128)
    e = K_.Int4Weight(*(t[None] for t in w))
    full = _rnd(g, 1, 128, 128)
    ids, wts = torch.empty(0, 1, dtype=torch.int32, device=cuda_dev), torch.empty(0, 1, device=cuda_dev)
    assert K_.linear_w4(x, w).shape == K_.decode_fwd_w4(x, w, None, w, None, w, None).shape == (0, 128)
    assert K_.moe_decode_fwd(x, ids, wts, full, full, full).shape == (0, 128)
    assert K_.moe_decode_fwd_w4(x, ids, wts, e, e, e).shape == (0, 128)
    i, p = K_.moe_route(x, full[0], 2)
    assert i.shape == p.shape == (0, 2)
    m = pkg.FusedMoEGatedMLP(128, 128, 4, 2).to(cuda_dev, BF)
    with torch.no_grad():
        assert m(x).shape == (0, 128) and m(x.view(2, 0, 128)).shape == (2, 0, 128)


def test_refusals(pkg, cuda_dev):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, 1)
    x, w, w64 = _rnd(g, 2, 128), _w4(pkg, g, 128, 128), _w4(pkg, g, 128, 128, group=64)
    full = _rnd(g, 3, 128, 128)
    ids, wts = _choices(g, 2, 3, 2)
    for call in (lambda: K_.linear_w4(_rnd(g, 65, 128), w), lambda: K_.linear_w4(_rnd(g, 2, 64), w),
                 lambda: K_.linear_w4(x[0], w), lambda: K_.linear_w4(x, w, bias=x[0, :64]),
                 lambda: K_.linear_w4(x, w, residual=x[:1]), lambda: K_.linear_w4(x, w._replace(scale=w.scale.t())),
                 lambda: K_.linear_w4(x, w._replace(scale=w.scale.half())),
                 lambda: K_.linear_w4(x, w._replace(zero=w.zero.to(torch.int32))),
                 lambda: K_.linear_w4(x, w._replace(w4=w.w4.view(torch.int8))),
                 lambda: K_.decode_fwd_w4(x, w, None, w64, None, w, None),
                 lambda: K_.decode_fwd_w4(x, w, None, w._replace(zero=None), None, w, None),
                 lambda: K_.decode_fwd_w4(x, w, x[0, :5], w, None, w, None),
                 lambda: K_.moe_route(x, full[0], 0), lambda: K_.moe_route(x, full[0, :3], 4),
                 lambda: K_.moe_route(x, full[0, :, :64], 2), lambda: K_.moe_route(_rnd(g, 2, 100), _rnd(g, 4, 96), 1),
                 lambda: K_.moe_decode_fwd(x, ids.long(), wts, full, full, full),
                 lambda: K_.moe_decode_fwd(x, ids, wts.half(), full, full, full),
                 lambda: K_.moe_decode_fwd(x, ids[:1], wts, full, full, full),
                 lambda: K_.moe_decode_fwd(x, ids, wts[:, :1], full, full, full),
                 lambda: K_.moe_decode_fwd(x, ids, wts, full, full[:2], full),
                 lambda: K_.moe_decode_fwd(_rnd(g, 2, 96), ids, wts, *(_rnd(g, 3, 96, 96) for _ in range(3))),
                 lambda: K_.moe_decode_fwd_w4(x, ids, wts, w, w, w)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: K_.linear_w4(x.float(), w), lambda: K_.moe_route(x.float(), full[0].float(), 1),
                 lambda: K_.moe_decode_fwd(x.float(), ids, wts, *(full.float(),) * 3)):
        with pytest.raises(NotImplementedError):
            call()
    cpu = K_.Int4Weight(*(t.cpu() for t in w))
    for call in (lambda: K_.linear_w4(x, cpu), lambda: K_.linear_w4(x, w._replace(scale=cpu.scale)),
                 lambda: K_.linear_w4(x, w._replace(zero=cpu.zero)),
                 lambda: K_.decode_fwd_w4(x, w, None, w, None, cpu, None),
                 lambda: K_.moe_decode_fwd(x, ids.cpu(), wts, full, full, full)):
        with pytest.raises(pkg._lib.GmlpError, match="no CPU path"):
            call()
    # a router row of 100 columns is no multiple of 8; 4-bit words have to start on 16 bytes
    with pytest.raises(pkg._lib.GmlpError, match="multiple of 8"):
        K_.moe_route(_rnd(g, 2, 100), _rnd(g, 4, 100), 1)
    buf = torch.zeros(128 * 64 + 8, dtype=torch.uint8, device=cuda_dev)[8:].view(128, 64)
    with pytest.raises(pkg._lib.GmlpError, match="aligned"):
        K_.linear_w4(x, w._replace(w4=buf))


# ------------------------------------------------------------ bad numbers --
@pytest.mark.parametrize("M", [3, 4, 6, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_bad_activations_stay_in_their_token(pkg, cuda_dev, M, bad):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    K, N, E, k = 512, 384, 5, 2
    x = _rnd(g, M, K)
    y = x.clone()
    y[1, 77] = bad
    wl = _w4(pkg, g, 200, K)
    dense = [_w4(pkg, g, *s) for s in ((N, K), (N, K), (K, N))]
    experts = [_rnd(g, E, *s, std=s[1] ** -0.5) for s in ((N, K), (N, K), (K, N))]
    experts4 = [K_.quantize_weight_int4(w, 128) for w in experts]
    ids, wts = _choices(g, M, E, k)
    rest = [m for m in range(M) if m != 1]
    for name, call in {
        "linear": lambda v: K_.linear_w4(v, wl), "mlp": lambda v: K_.decode_fwd_w4(v, dense[0], None, dense[1], None, dense[2], None),
        "moe": lambda v: K_.moe_decode_fwd(v, ids, wts, *experts),
        "moe_w4": lambda v: K_.moe_decode_fwd_w4(v, ids, wts, *experts4),
    }.items():
        a, b = call(x), call(y)
        assert torch.equal(a[rest], b[rest]), name
        assert not torch.isfinite(b[1]).any(), name


def test_router_on_bad_numbers_and_ties(pkg, cuda_dev):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, 5)
    for E, k in ((6, 6), (40, 8), (128, 8), (300, 32), (512, 32)):
        x, w = _rnd(g, 5, 256), _rnd(g, E, 256, std=0.06)
        x[1, 3], x[2] = float("nan"), float("inf")
        x[3] = 0                                      # every logit equal: the first k experts, equal weights
        w[E // 2] = w[E // 3]                         # two equal logits: the lower index first
        ids, wts = K_.moe_route(x, w, k)
        for t in range(5):
            row = ids[t].tolist()
            assert len(set(row)) == k and all(0 <= e < E for e in row)
        assert ids[3].tolist() == list(range(k)) and ((wts[3] * k - 1).abs() <= 2.0 ** -20).all()
        want_ids, want = ft.route(x[[0, 4]], w, k, True)
        assert torch.equal(ids[[0, 4]], want_ids)
        assert ((wts[[0, 4]].double() - want).abs() <= want * 2.0 ** -17).all()
    # only one expert's logit is a NaN: it is the last choice
    x, w = _rnd(g, 2, 64), _rnd(g, 9, 64)
    w[4, 0] = float("nan")
    ids, _ = K_.moe_route(x, w, 8)
    assert not (ids == 4).any()
    ids, _ = K_.moe_route(x, w, 9)
    assert (ids[:, 8] == 4).all()


@pytest.mark.parametrize("scale", [1e-7, 1e4])
def test_small_and_large_activations(pkg, cuda_dev, scale):
    """A power of two per group or token carries any magnitude of the type."""
    g = _gen(cuda_dev, 2)
    for M in (2, 30):
        for dt in (BF, FP):
            w = _w4(pkg, g, 300, 512, dt=dt)
            x = _rnd(g, M, 512, std=scale, dt=dt)
            x[0, :200] *= 1e-3
            y = pkg.ops.kernels.linear_w4(x, w)
            ft.check(y, *ft.linear(x, ft.unpack(*w), None, None, dt, 128), f"M={M} scale={scale}")


# ------------------------------------------------------ ends of the ranges --
@pytest.mark.parametrize("M,rows", [(2, 131072), (7, 131075), (3, 131073)])
def test_weights_past_32_bit_offsets(pkg, cuda_dev, M, rows):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    cols, group = 65536 + 256, 128
    w4 = torch.randint(0, 256, (rows, cols // 2), dtype=torch.uint8, device=cuda_dev, generator=g)
    scale = (torch.rand((cols // group, rows), device=cuda_dev, generator=g) * 2.0 ** -10 + 2.0 ** -12).to(BF)
    zero = torch.randint(0, 16, (cols // group, rows), dtype=torch.uint8, device=cuda_dev, generator=g)
    assert w4.numel() > 2 ** 32
    x = _rnd(g, M, cols)
    y = K_.linear_w4(x, K_.Int4Weight(w4, scale, zero))
    for lo in (0, 65000, rows - 260):
        part = slice(lo, lo + 260)
        w = ft.unpack(w4[part], scale[:, part], zero[:, part])
        ft.check(y[:, part], *ft.linear(x, w, None, None, BF, group), f"rows {lo}..")


@pytest.mark.parametrize("four_bit", [False, True])
def test_experts_past_32_bit_offsets(pkg, cuda_dev, four_bit):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, 9)
    E, K, N, T, k = 512, 4096, 2176, 3, 2
    ids = torch.tensor([[511, 3], [0, 511], [509, 260]], dtype=torch.int32, device=cuda_dev)
    wts = torch.tensor([[0.75, 0.25], [0.5, 0.5], [0.125, 0.5]], device=cuda_dev)
    chosen = sorted(set(ids.flatten().tolist()))
    small = torch.tensor([[chosen.index(e) for e in row] for row in ids.tolist()], dtype=torch.int32, device=cuda_dev)
    x = _rnd(g, T, K)
    if four_bit:
        ws = []
        for r, c in ((N, K), (N, K), (K, N)):
            q = torch.randint(0, 256, (E, r, c // 2), dtype=torch.uint8, device=cuda_dev, generator=g)
            s = (torch.rand((E, c // 128, r), device=cuda_dev, generator=g) * 2.0 ** -9 + 2.0 ** -12).to(BF)
            z = torch.randint(0, 16, s.shape, dtype=torch.uint8, device=cuda_dev, generator=g)
            ws.append(K_.Int4Weight(q, s, z))
        y = K_.moe_decode_fwd_w4(x, ids, wts, *ws)
        full = [ft.unpack(w.w4[chosen], w.scale[chosen], w.zero[chosen]) for w in ws]
        group = 128
    else:
        ws = [torch.empty((E, r, c), dtype=BF, device=cuda_dev).normal_(0, c ** -0.5, generator=g)
              for r, c in ((N, K), (N, K), (K, N))]
        assert ws[0].numel() > 2 ** 32
        y = K_.moe_decode_fwd(x, ids, wts, *ws)
        full, group = [w[chosen].double() for w in ws], 0
    ft.check(y, *ft.moe(x, small, wts, *full, None, BF, group=group), "experts past 32 bits")


@pytest.mark.parametrize("four_bit", [False, True])
def test_widest_routing_table(pkg, cuda_dev, four_bit):
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, 4)
    T, E, k, K, N = 64, 512, 32, 64, 64
    x = _rnd(g, T, K)
    ids, wts = _choices(g, T, E, k)
    ws = [_rnd(g, E, *s, std=s[1] ** -0.5) for s in ((N, K), (N, K), (K, N))]
    if four_bit:
        packed = [K_.quantize_weight_int4(w, 32) for w in ws]
        y = K_.moe_decode_fwd_w4(x, ids, wts, *packed)
        ws = [ft.unpack(*w) for w in packed]
    else:
        y = K_.moe_decode_fwd(x, ids, wts, *ws)
        ws = [w.double() for w in ws]
    ft.check(y, *ft.moe(x, ids, wts, *ws, None, BF, group=32 if four_bit else 0), "512 experts, 32 choices")


# ------------------------------------------------------------- modules --
@pytest.mark.parametrize("tokens", [(1,), (2, 3), (64,), (5, 20), (130,)])
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dt", [BF, FP])
def test_moe_module(pkg, cuda_dev, tokens, bits, dt):
    torch.manual_seed(sum(tokens))
    m = pkg.FusedMoEGatedMLP(256, 384, 10, 3, hidden_act="gelu", renormalize=bits == 4).to(cuda_dev, dt)
    g = _gen(cuda_dev, 8)
    x = _rnd(g, *tokens, 256, dt=dt)
    res = _rnd(g, *tokens, 256, dt=dt)
    ws, group = [m.gate_proj, m.up_proj, m.down_proj], 0
    if bits == 4:
        m.quantize_decode_weights(group_size=64)
        ws, group = [ft.unpack(*w) for w in m._w4], 64
    with torch.no_grad():
        y, z = m(x, residual=res), m(x)
        assert y.shape == z.shape == x.shape
        rows, r = x.view(-1, 256), res.view(-1, 256)
        ids, wts = pkg.ops.kernels.moe_route(rows, m.router.weight, 3, m.renormalize)
        assert torch.equal(ids, ft.route(rows, m.router.weight, 3, m.renormalize)[0])
        for lo in range(0, rows.shape[0], 64):
            p = slice(lo, lo + 64)
            args = (rows[p], ids[p], wts[p], *(w.double() for w in ws))
            ft.check(y.view(-1, 256)[p], *ft.moe(*args, r[p], dt, "gelu", group), "module with residual")
            ft.check(z.view(-1, 256)[p], *ft.moe(*args, None, dt, "gelu", group), "module")


@pytest.mark.parametrize("M", [1, 8, 64])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_dense_module_on_four_bits(pkg, cuda_dev, M, group):
    torch.manual_seed(M)
    m = pkg.FusedGatedMLP(256, 384, hidden_act="silu").to(cuda_dev, BF)
    g = _gen(cuda_dev, M)
    x = _rnd(g, M, 256)
    many = _rnd(g, 65, 256)
    with torch.no_grad():
        plain, plain_many = m(x), m(many)
        m.quantize_decode_weights(bits=4, group_size=group)
        y = m(x, residual=x)
        q = [ft.unpack(*w) for w in m._w4]
        ft.check(y, *ft.mlp(x, q[0], m.gate_proj.bias, q[1], m.up_proj.bias, q[2], m.down_proj.bias, x, BF, "silu", group),
                 "module on 4-bit weights")
        assert torch.equal(m(many), plain_many)       # more than 64 tokens: the 16-bit weights
        m.quantize_decode_weights()                   # 8 bits in their place, and none again
        assert m._w4 is None
        m.quantize_decode_weights(False)
        assert torch.equal(m(x), plain)
    m.quantize_decode_weights(bits=4, group_size=group)
    m(x).sum().backward()                             # training still sees the 16-bit weights
    assert m.gate_proj.weight.grad is not None


@pytest.mark.parametrize("M", [1, 6, 64])
def test_a_decoder_step_of_all_of_them(pkg, cuda_dev, M):
    """A dense 4-bit block, a mixture in 16 bits, a mixture in 4 bits and a 4-bit vocabulary projection, one after the other:
    eagerly stage by stage against the restatement, then captured and replayed on new inputs, with the eager call's bits."""
    torch.manual_seed(M)
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    H = 512
    dense = pkg.FusedGatedMLP(H, 896, bias=False).to(cuda_dev, BF)
    dense.quantize_decode_weights(bits=4)
    moe, moe4 = (pkg.FusedMoEGatedMLP(H, 256, 16, 4).to(cuda_dev, BF) for _ in range(2))
    moe4.quantize_decode_weights()
    vocab = _w4(pkg, g, 5003, H)

    def step(x):
        a = dense(x, residual=x)
        b = moe(a, residual=a)
        c = moe4(b, residual=b)
        return a, b, c, K_.linear_w4(c, vocab)

    with torch.no_grad():
        x = _rnd(g, M, H)
        a, b, c, y = step(x)
        q = [ft.unpack(*w) for w in dense._w4]
        ft.check(a, *ft.mlp(x, q[0], None, q[1], None, q[2], None, x, BF, "silu", 128), "dense")
        for name, inp, out, m in (("moe", a, b, moe), ("moe4", b, c, moe4)):
            ids, wts = K_.moe_route(inp, m.router.weight, 4)
            four = m._w4 is not None
            ws = [ft.unpack(*w) for w in m._w4] if four else [m.gate_proj.double(), m.up_proj.double(), m.down_proj.double()]
            ft.check(out, *ft.moe(inp, ids, wts, *ws, inp, BF, group=128 if four else 0), name)
        ft.check(y, *ft.linear(c, ft.unpack(*vocab), None, None, BF, 128), "vocabulary")
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(static)
        for _ in range(4):
            x = _rnd(g, M, H)
            static.copy_(x)
            graph.replay()
            for got, want in zip(out, step(x)):
                assert torch.equal(got, want)


@pytest.mark.parametrize("M", [1, 5, 64])
def test_while_another_kernel_holds_most_sms(pkg, cuda_dev, M):
    """A long GEMM holds 100 SMs, so that only some blocks of a call are there at a time: those leave their shares of the
    cut tiles to the ones that come later, and the results keep their bits."""
    K_ = pkg.ops.kernels
    lib = pkg._lib.load()
    g = _gen(cuda_dev, M)
    K, N, E, k = 2048, 4096, 8, 2
    x, xl = _rnd(g, M, K), _rnd(g, M, 8192)
    wl = _w4(pkg, g, 2048, 8192)
    dense = [_w4(pkg, g, *s) for s in ((N, K), (N, K), (K, N))]
    experts = [_rnd(g, E, *s, std=s[1] ** -0.5) for s in ((N, K), (N, K), (K, N))]
    experts4 = [K_.quantize_weight_int4(w, 128) for w in experts]
    ids, wts = _choices(g, M, E, k)
    calls = [lambda: K_.linear_w4(xl, wl), lambda: K_.decode_fwd_w4(x, dense[0], None, dense[1], None, dense[2], None),
             lambda: K_.moe_decode_fwd(x, ids, wts, *experts), lambda: K_.moe_decode_fwd_w4(x, ids, wts, *experts4)]
    want = [c() for c in calls]
    a = _rnd(g, 16384, 16384)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    before = lib.gmlp_set_sm_limit(100)
    try:
        with torch.cuda.stream(side):
            K_.gemm(a, a)
            torch.cuda.synchronize()
            started, done = torch.cuda.Event(), torch.cuda.Event()
            started.record()
            for _ in range(4):
                K_.gemm(a, a)
            done.record()
    finally:
        lib.gmlp_set_sm_limit(before)
    started.synchronize()
    got = [c() for _ in range(5) for c in calls]
    mine = torch.cuda.Event()
    mine.record()
    mine.synchronize()
    assert not done.query()                           # the GEMMs outlast the calls
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(calls)]), i


@pytest.mark.parametrize("M", [2, 9, 50])
@pytest.mark.parametrize("shift", [2, 6, 12])
def test_scales_and_zeros_on_any_four_byte_boundary(pkg, cuda_dev, M, shift):
    """Views that start inside a 16-byte block, with and without zeros: the same bits as aligned copies."""
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    for rows in (256, 333):
        for symmetric in (False, True):
            w = _w4(pkg, g, rows, 512, group=64, symmetric=symmetric)
            x = _rnd(g, M, 512)
            s = torch.empty(w.scale.numel() + shift, dtype=BF, device=cuda_dev)[shift:].view(w.scale.shape).copy_(w.scale)
            z = None if symmetric else torch.empty(w.zero.numel() + 2 * shift, dtype=torch.uint8,
                                                   device=cuda_dev)[2 * shift:].view(w.zero.shape).copy_(w.zero)
            y = K_.linear_w4(x, K_.Int4Weight(w.w4, s, z))
            assert torch.equal(y, K_.linear_w4(x, w))
            ft.check(y, *ft.linear(x, ft.unpack(*w), None, None, BF, 64), "shifted scales")


@pytest.mark.parametrize("M", [1, 4, 8, 64])
@pytest.mark.parametrize("largest", [3e38, 1e30, 1e-33])
def test_ends_of_bfloat16(pkg, cuda_dev, M, largest):
    """Activations next to the type's largest number whose products with the weights are finite, and tiny ones."""
    K_ = pkg.ops.kernels
    g = _gen(cuda_dev, M)
    w = _w4(pkg, g, 300, 256, group=64)
    w = w._replace(scale=(w.scale.float() * 2.0 ** -6).to(BF))
    x = ((torch.rand((M, 256), generator=g, device=cuda_dev) * 2 - 1) * largest).to(BF)
    y = K_.linear_w4(x, w)
    assert torch.isfinite(y).all()
    ft.check(y, *ft.linear(x, ft.unpack(*w), None, None, BF, 64), f"M={M} largest={largest}")


@pytest.mark.parametrize("M", [2, 12])
def test_dense_module_with_sizes_only_four_bits_take(pkg, cuda_dev, M):
    torch.manual_seed(M)
    m = pkg.FusedGatedMLP(96, 160, bias=False).to(cuda_dev, BF)
    m.quantize_decode_weights(bits=4, group_size=32)
    x = _rnd(_gen(cuda_dev, M), M, 96)
    q = [ft.unpack(*w) for w in m._w4]
    with torch.no_grad():
        ft.check(m(x), *ft.mlp(x, q[0], None, q[1], None, q[2], None, None, BF, "silu", 32), "96 x 160")


def test_two_host_threads_on_one_stream(pkg, cuda_dev):
    """Their kernels interleave on the stream: each thread has work buffers of its own."""
    import threading

    sets = [_calls(pkg, cuda_dev, M, seed=3 * M) for M in (5, 40)]
    want = [{n: c() for n, c in s.items()} for s in sets]
    bad = []

    def run(calls, expected):
        for _ in range(100):
            for n, c in calls.items():
                if not torch.equal(c(), expected[n]):
                    bad.append(n)

    threads = [threading.Thread(target=run, args=a) for a in zip(sets, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
