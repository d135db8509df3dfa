"""Measured cases of the few-token serving operators: products with 4-bit weights and group scales, the gated MLP on
such weights, and mixture-of-experts layers (router and experts, 16-bit and 4-bit) for 1 to 64 tokens.

4-bit format: a row of `cols` weights is cols / 8 little-endian 32-bit words; word j holds columns 8j .. 8j+7, column
8j + c as an unsigned nibble at bit SHIFTS[c]. w = (q - zero) * scale with one scale (x's type) and one zero (0..15,
8 where there are none) for each group of `group` columns of a row, both stored [cols / group, rows].
"""
import math

import torch

own = False

SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token through a square projection of an 8B-class block: the smallest call, latency counts
        dict(name="w4_linear_m1_4096x4096", op="linear", M=1, K=4096, N=4096, group=128, zeros=True, bias=False,
             residual=False, dtype="bf16"),
        # a vocabulary projection for a batch of eight sequences
        dict(name="w4_linear_m8_131072x4096", op="linear", M=8, K=4096, N=131072, group=128, zeros=True, bias=False,
             residual=False, dtype="bf16"),
        # odd everything: tokens, rows and columns that fill no tile, the finest groups, symmetric, bias and residual
        dict(name="w4_linear_m17_5001x2080", op="linear", M=17, K=2080, N=5001, group=32, zeros=False, bias=True,
             residual=True, dtype="fp16"),
        # the decode configuration of the benchmark (K=8192, N=28672), one token and a full batch
        dict(name="w4_mlp_m1_k8192_n28672", op="mlp", M=1, K=8192, N=28672, group=128, zeros=True, bias=False,
             residual=False, act="silu", dtype="bf16"),
        dict(name="w4_mlp_m64_k8192_n28672", op="mlp", M=64, K=8192, N=28672, group=128, zeros=True, bias=False,
             residual=True, act="silu", dtype="fp16"),
        # the 8B block of the benchmark at a medium batch, groups of 64
        dict(name="w4_mlp_m16_k4096_n14336", op="mlp", M=16, K=4096, N=14336, group=64, zeros=False, bias=False,
             residual=True, act="silu", dtype="bf16"),
        # a small block with biases and another activation
        dict(name="w4_mlp_m3_k512_n896", op="mlp", M=3, K=512, N=896, group=128, zeros=True, bias=True,
             residual=False, act="gelu", dtype="fp16"),
        # few large experts, one token: two experts are streamed
        dict(name="moe_t1_e8_k2_4096x14336", op="moe", M=1, E=8, top_k=2, K=4096, N=14336, renormalize=True,
             residual=True, act="silu", dtype="bf16"),
        # many small experts, a full batch: every expert is streamed
        dict(name="moe_t64_e64_k6_2048x1408", op="moe", M=64, E=64, top_k=6, K=2048, N=1408, renormalize=False,
             residual=False, act="silu", dtype="fp16"),
        # a small ragged layer
        dict(name="moe_t5_e18_k3_576x320", op="moe", M=5, E=18, top_k=3, K=576, N=320, renormalize=True,
             residual=True, act="silu", dtype="bf16"),
        # 4-bit experts: one token of a fine-grained mixture, and a batch over wider experts
        dict(name="moe_w4_t1_e128_k8_2048x768", op="moe_w4", M=1, E=128, top_k=8, K=2048, N=768, group=128,
             zeros=True, renormalize=True, residual=True, act="silu", dtype="bf16"),
        dict(name="moe_w4_t32_e32_k4_4096x1792", op="moe_w4", M=32, E=32, top_k=4, K=4096, N=1792, group=64,
             zeros=False, renormalize=True, residual=False, act="silu", dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "mlp", "moe", "moe_w4"))
    c = dict(op=op, M=_log(rng, 1, 64), dtype=rng.choice(("bf16", "fp16")), residual=rng.random() < 0.5)
    if op in ("linear", "mlp", "moe_w4"):
        c.update(group=rng.choice((32, 64, 128)), zeros=rng.random() < 0.5)
    if op == "linear":
        c.update(K=c["group"] * _log(rng, 256 // c["group"], 8192 // c["group"]), N=_log(rng, 250, 65000),
                 bias=rng.random() < 0.5)
    elif op == "mlp":
        c.update(K=c["group"] * _log(rng, 256 // c["group"], 8192 // c["group"]),
                 N=c["group"] * _log(rng, 512 // c["group"], 28672 // c["group"]), bias=rng.random() < 0.5,
                 act=rng.choice(("silu", "gelu", "relu")))
    else:
        step = c["group"] if op == "moe_w4" else 64
        c.update(E=_log(rng, 4, 128), K=step * _log(rng, 256 // step, 4096 // step), renormalize=rng.random() < 0.5,
                 act="silu")
        c["top_k"] = rng.randint(1, min(8, c["E"]))
        most = min(14336, 400_000_000 // (c["E"] * c["K"]))  # all experts together no larger than the largest listed
        c["N"] = step * max(1, _log(rng, 256 // step, max(256, most) // step))
    return c


# ---------------------------------------------------------------------------------------------------- inputs --
def _int4(w, group, zeros, dtype):
    """Weights [.., rows, cols] (float32) in the 4-bit format: (uint8 words, scale, zero or None)."""
    v = w.unflatten(-1, (-1, group))
    if zeros:
        lo, hi = v.amin(-1).clamp_max(0), v.amax(-1).clamp_min(0)
        scale = ((hi - lo) / 15).clamp_min(1e-8).to(dtype)
        zero = (-lo / scale.float()).round().clamp(0, 15)
    else:
        scale = (v.abs().amax(-1) / 7.5).clamp_min(1e-8).to(dtype)
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    q = (v / scale.float()[..., None]).round().add_(zero[..., None]).clamp_(0, 15).to(torch.int32).flatten(-2)
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device=w.device)
    words = (q.unflatten(-1, (-1, 8)) << shifts).sum(-1).to(torch.int32)
    return (words.view(torch.uint8), scale.transpose(-1, -2).contiguous(),
            zero.to(torch.uint8).transpose(-1, -2).contiguous() if zeros else None)


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=dev).mul_(std)

    M, K, N = case["M"], case["K"], case["N"]
    x = rnd(M, K)
    x = (x * (1 + 7 * (torch.rand((K,), generator=g, device=dev) < 0.01))).to(dt)  # a few outlier channels
    s = {"case": case, "x": x}
    out = N if case["op"] == "linear" else K
    s["residual"] = rnd(M, out).to(dt) if case["residual"] else None
    if case["op"] == "linear":
        s["w"] = _int4(rnd(N, K, std=K ** -0.5), case["group"], case["zeros"], dt)
        s["bias"] = rnd(N).to(dt) if case["bias"] else None
        return s
    E = (case["E"],) if "E" in case else ()
    w = []
    for shape, std in (((N, K), K ** -0.5), ((N, K), K ** -0.5), ((K, N), N ** -0.5)):
        full = rnd(*E, *shape, std=std)
        w.append(full.to(dt) if case["op"] == "moe" else _int4(full, case["group"], case["zeros"], dt))
        del full
    s["w_gate"], s["w_up"], s["w_down"] = w
    if case["op"] == "mlp":
        s["b_gate"], s["b_up"], s["b_down"] = (rnd(n, std=0.5).to(dt) if case["bias"] else None for n in (N, N, K))
    else:
        s["w_router"] = rnd(case["E"], K, std=1.5 * K ** -0.5).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ plain forms --
def _dequant(w):
    words, scale, zero = w
    shifts = torch.tensor(SHIFTS, dtype=torch.int32, device=words.device)
    q = ((words.view(torch.int32)[..., None] >> shifts) & 15).flatten(-2).float()
    scale = scale.transpose(-1, -2).float()
    zero = 8.0 if zero is None else zero.transpose(-1, -2).float()[..., None]
    return ((q.unflatten(-1, (scale.shape[-1], -1)) - zero) * scale[..., None]).flatten(-2)


def _act(name, v):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    return v * (v > 0)


def _plus(v, t):
    return v if t is None else v + t.float()


def _plain_linear(s):
    y = s["x"].float() @ _dequant(s["w"]).t()
    return _plus(_plus(y, s["bias"]), s["residual"]).to(s["x"].dtype)


def _plain_mlp(s):
    x = s["x"].float()
    gate = _plus(x @ _dequant(s["w_gate"]).t(), s["b_gate"])
    up = _plus(x @ _dequant(s["w_up"]).t(), s["b_up"])
    y = (_act(s["case"]["act"], gate) * up) @ _dequant(s["w_down"]).t()
    return _plus(_plus(y, s["b_down"]), s["residual"]).to(s["x"].dtype)


def _plain_moe(s):
    c, x = s["case"], s["x"].float()
    logits = s["x"].double() @ s["w_router"].double().t()  # 64 bits: the choice of experts lies next to a border
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    p, ids = p[:, : c["top_k"]], ids[:, : c["top_k"]]
    p = (p / p.sum(-1, keepdim=True) if c["renormalize"] else p).float()
    if c["M"] * c["top_k"] <= c["E"]:  # each choice's weights gathered
        def of(w):
            w = tuple(None if t is None else t[ids] for t in w) if c["op"] == "moe_w4" else w[ids]
            return _dequant(w) if c["op"] == "moe_w4" else w.float()

        v = x[:, None, :, None]
        h = _act(c["act"], of(s["w_gate"]) @ v) * (of(s["w_up"]) @ v)
        y = ((of(s["w_down"]) @ h)[..., 0] * p[..., None]).sum(1)
    else:  # fewer bytes: every expert once, with a weight of zero where a token did not choose it
        def of(w):
            return _dequant(w) if c["op"] == "moe_w4" else w.float()

        share = torch.zeros((c["M"], c["E"]), device=x.device).scatter_(1, ids, p).t()[..., None]
        h = _act(c["act"], x @ of(s["w_gate"]).transpose(1, 2)) * (x @ of(s["w_up"]).transpose(1, 2))
        y = ((h * share) @ of(s["w_down"]).transpose(1, 2)).sum(0)
    return {"y": _plus(y, s["residual"]).to(s["x"].dtype), "ids": ids.to(torch.int32), "weights": p}


# ---------------------------------------------------------------------------------------- the framework's calls --
def _own(s):
    from triton_gated_mlp_b200.ops import kernels as k

    c, x = s["case"], s["x"]
    if c["op"] == "linear":
        return k.linear_w4(x, k.Int4Weight(*s["w"]), bias=s["bias"], residual=s["residual"])
    if c["op"] == "mlp":
        return k.decode_fwd_w4(x, k.Int4Weight(*s["w_gate"]), s["b_gate"], k.Int4Weight(*s["w_up"]), s["b_up"],
                               k.Int4Weight(*s["w_down"]), s["b_down"], act=c["act"], residual=s["residual"])
    ids, weights = k.moe_route(x, s["w_router"], c["top_k"], renormalize=c["renormalize"])
    if c["op"] == "moe":
        y = k.moe_decode_fwd(x, ids, weights, s["w_gate"], s["w_up"], s["w_down"], act=c["act"],
                             residual=s["residual"])
    else:
        y = k.moe_decode_fwd_w4(x, ids, weights, k.Int4Weight(*s["w_gate"]), k.Int4Weight(*s["w_up"]),
                                k.Int4Weight(*s["w_down"]), act=c["act"], residual=s["residual"])
    return {"y": y, "ids": ids, "weights": weights}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "linear":
        return _plain_linear(state)
    if op == "mlp":
        return _plain_mlp(state)
    return _plain_moe(state)


# --------------------------------------------------------------------------------------------------- the work --
def work(case):
    M, K, N, op = case["M"], case["K"], case["N"], case["op"]
    each = 0.5 + (2 + (1 if case["zeros"] else 0)) / case["group"] if "group" in case else 2.0  # bytes of a weight
    out = N if op == "linear" else K
    act = 2 * M * (K + out + (out if case["residual"] else 0))
    if op == "linear":
        return {"bytes": each * K * N + act + (2 * N if case["bias"] else 0), "flops": 2.0 * M * K * N}
    if op == "mlp":
        return {"bytes": each * 3 * K * N + act + (2 * (2 * N + K) if case["bias"] else 0), "flops": 6.0 * M * K * N}
    E, k = case["E"], case["top_k"]
    active = E * (1 - (1 - k / E) ** M)  # experts that M tokens reach between them, on average over the inputs
    return {"bytes": each * 3 * K * N * active + 2 * E * K + act + 8 * M * k,
            "flops": 6.0 * M * k * K * N + 2.0 * M * E * K}


# ------------------------------------------------------------------------------------- from the definition, 64 bits --
def _weights64(w):
    if not isinstance(w, tuple):
        return w.double()
    words, scale, zero = w
    b = words.unflatten(-1, (-1, 4))
    q = torch.empty((*b.shape[:-1], 8), dtype=torch.float64, device=b.device)
    q[..., 0::4], q[..., 2::4] = (b & 15)[..., 0:2].double(), (b >> 4)[..., 0:2].double()
    q[..., 1::4], q[..., 3::4] = (b & 15)[..., 2:4].double(), (b >> 4)[..., 2:4].double()
    q = q.flatten(-2)
    group = q.shape[-1] // scale.shape[-2]
    by_column = lambda t: t.double().repeat_interleave(group, dim=-2).transpose(-1, -2)  # noqa: E731
    return (q - (8.0 if zero is None else by_column(zero))) * by_column(scale)


def _act64(name, v):
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}
    return f[name](v)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    res = 0 if s["residual"] is None else s["residual"].double()
    if case["op"] == "linear":
        return torch.einsum("mk,nk->mn", x, _weights64(s["w"])) + (0 if s["bias"] is None else s["bias"].double()) + res
    if case["op"] == "mlp":
        b = [0 if s[n] is None else s[n].double() for n in ("b_gate", "b_up", "b_down")]
        g = torch.einsum("mk,nk->mn", x, _weights64(s["w_gate"])) + b[0]
        u = torch.einsum("mk,nk->mn", x, _weights64(s["w_up"])) + b[1]
        return torch.einsum("mn,kn->mk", _act64(case["act"], g) * u, _weights64(s["w_down"])) + b[2] + res
    p = torch.softmax(torch.einsum("mk,ek->me", x, s["w_router"].double()), -1)
    order = torch.argsort(-p, dim=-1, stable=True)[:, : case["top_k"]]
    chosen = torch.gather(p, 1, order)
    if case["renormalize"]:
        chosen = chosen / chosen.sum(1, keepdim=True)
    y = torch.zeros_like(x) + res
    one = lambda w, e: _weights64(tuple(None if t is None else t[e] for t in w) if isinstance(w, tuple) else w[e])  # noqa: E731
    for e in range(case["E"]):
        token, place = torch.nonzero(order == e, as_tuple=True)
        if len(token):
            v = x[token]
            h = _act64(case["act"], v @ one(s["w_gate"], e).t()) * (v @ one(s["w_up"], e).t())
            y.index_add_(0, token, (h @ one(s["w_down"], e).t()) * chosen[token, place][:, None])
    return {"y": y, "ids": None, "weights": chosen}
