"""The decoder-layer operators, as they are used: cases, their plain forms and their exact values.

``rope``    rotary positions of queries and keys (``ops.rope``; with gradients ``train.rope``)
``linear``  matrix product with bias, activation and residual (``ops.linear_residual``; with gradients ``train.linear_residual``)
``moe``     the whole expert layer for a few tokens (``str_backbone.moe_few``)

``own`` False computes the plain forms from elementary torch operations in 32 bits, True calls the library."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
PRECISION = {"fp32": "fp32", "bf16": "bf16", "fp16": "f16"}        # the library's names of the weight forms
ACTS = ("none", "relu", "gelu_erf", "gelu_tanh", "leaky", "silu", "tanh")     # in the order of the library's ACT_* codes


def listed():
    return [
        # one new token of eight scenarios in a 16-head decoder of width 1024: the key-point loop, where latency is all
        dict(name="rope_one_token", op="rope", type="bf16", batch=8, seq=1, heads=16, kv_heads=8, width=64, part=64, layout="half", theta=1e6,
             factor=1.0, far=900, grad=False),
        # a long prefill, the width-128 heads of the large decoders: memory bound
        dict(name="rope_prefill", op="rope", type="bf16", batch=8, seq=4096, heads=32, kv_heads=8, width=128, part=128, layout="half", theta=1e6,
             factor=1.0, far=4096, grad=False),
        # a training step over packed tokens of odd length: part of the head, neighbouring pairs, frequencies scaled for far positions
        dict(name="rope_train_far", op="rope", type="fp16", batch=3, seq=1747, heads=16, kv_heads=4, width=96, part=48, layout="interleaved",
             theta=1e4, factor=8.0, far=1000000, grad=True),
        # out-projection of one token
        dict(name="linear_one_token", op="linear", type="bf16", rows=1, n=1024, k=1024, act="none", residual=True, grad=False),
        # up-projection of the few tokens of a batch of scenarios
        dict(name="linear_few_tokens", op="linear", type="fp16", rows=24, n=6144, k=1536, act="silu", residual=False, grad=False),
        # prefill of eight scenarios with 873 context tokens each
        dict(name="linear_prefill", op="linear", type="bf16", rows=6984, n=4096, k=1024, act="gelu_tanh", residual=True, grad=False),
        # a training step of a wide layer, forward and backward
        dict(name="linear_train", op="linear", type="bf16", rows=8192, n=4096, k=4096, act="gelu_erf", residual=True, grad=True),
        # the same in fp32 at sizes that fill no tile
        dict(name="linear_train_odd", op="linear", type="fp32", rows=1037, n=1020, k=772, act="silu", residual=True, grad=True),
        # one token of the small wide decoder
        dict(name="moe_one_token", op="moe", type="bf16", tokens=1, d=512, inter=2048, experts=8, top_k=2),
        # a batch of eight scenarios, one token each, the medium decoder
        dict(name="moe_batch", op="moe", type="bf16", tokens=8, d=1024, inter=4096, experts=8, top_k=2),
        # as many tokens as the few-token form takes, the widest decoder: every expert is chosen
        dict(name="moe_64_tokens", op="moe", type="bf16", tokens=64, d=1536, inter=6144, experts=8, top_k=2),
        # fp32 weights of the small decoder, an odd batch
        dict(name="moe_fp32", op="moe", type="fp32", tokens=5, d=256, inter=1024, experts=8, top_k=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "linear", "linear", "moe"))
    kind = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "rope":
        width = rng.choice((32, 64, 80, 96, 128, 256))
        heads = rng.choice((4, 8, 12, 16, 32))
        kv = rng.choice([h for h in (1, 2, 4, 8) if heads % h == 0])
        batch, grad = _log(rng, 1, 32), rng.random() < 0.4
        per_token = (heads + kv) * width * SIZE[kind] * (2 if grad else 1)
        seq = _log(rng, 1, max(2, min(8192, 320_000_000 // (batch * per_token))))
        part = rng.choice((width, width // 2, 2 * rng.randint(1, width // 2)))
        return dict(op=op, type=kind, batch=batch, seq=seq, heads=heads, kv_heads=kv, width=width, part=part,
                    layout=rng.choice(("half", "interleaved")), theta=rng.choice((1e4, 5e5, 1e6)), factor=rng.choice((1.0, 4.0, 16.0)),
                    far=max(seq, _log(rng, 64, 2_000_000)), grad=grad)
    if op == "linear":
        grad = rng.random() < 0.5
        rows = _log(rng, 1, 64) if not grad and rng.random() < 0.5 else _log(rng, 64, 16384)
        step = rng.choice((1, 4, 8, 32, 64))
        n, k = (max(8, _log(rng, 64, 6144) // step * step) for _ in range(2))
        most = 1.0e11 if not grad else 2.5e11
        if kind == "fp32":
            most /= 4
        while 2.0 * rows * n * k > most:
            rows = max(1, rows // 2)
        return dict(op=op, type=kind, rows=rows, n=n, k=k, act=rng.choice(ACTS), residual=rng.random() < 0.7, grad=grad)
    experts = rng.choice((4, 8, 8, 16, 64))
    d, inter = 32 * _log(rng, 4, 48), 32 * _log(rng, 8, 192)
    while experts * 3 * d * inter * SIZE[kind] > 450_000_000:
        inter = max(64, inter // 64 * 32)
    return dict(op=op, type=kind, tokens=_log(rng, 1, 64), d=d, inter=inter, experts=experts, top_k=rng.choice([k for k in (1, 2, 2, 4, 6) if k <= experts]))


def _frequencies(part, theta, factor):
    """Radians a position of every rotated pair, 64 bits.  ``factor`` > 1: the slow pairs (less than one turn in 4096 positions) are
    slowed by the factor, the fast ones (more than 32 turns) are kept, those between are blended; the amplitude grows with it."""
    j = torch.arange(0, part, 2, dtype=torch.float64)
    w = theta ** (-j / part)
    if factor == 1.0:
        return w, 1.0
    turns = 4096 * w / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return w * keep + w / factor * (1 - keep), 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, kind=t):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return (x * scale).to(kind)

    s = dict(case)
    if case["op"] == "rope":
        B, S, W = case["batch"], case["seq"], case["width"]
        s["q"], s["k"] = normal(B, S, case["heads"], W), normal(B, S, case["kv_heads"], W)
        first = torch.randint(0, case["far"] - S + 1, (B, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(S, device="cuda")
        w, s["amplitude"] = _frequencies(case["part"], case["theta"], case["factor"])
        s["inv_freq"] = w.cuda()
        if case["grad"]:
            s["q"].requires_grad_()
            s["k"].requires_grad_()
            s["dq"], s["dk"] = normal(B, S, case["heads"], W), normal(B, S, case["kv_heads"], W)
    elif case["op"] == "linear":
        M, N, K = case["rows"], case["n"], case["k"]
        s["x"], s["w"], s["b"] = normal(M, K), normal(N, K, scale=K ** -0.5), normal(N, scale=0.5)
        s["res"] = normal(M, N) if case["residual"] else None
        if case["grad"]:
            for name in ("x", "w", "b", "res"):
                if s[name] is not None:
                    s[name].requires_grad_()
            s["dy"] = normal(M, N)
    else:
        T, d, inter, E = case["tokens"], case["d"], case["inter"], case["experts"]
        s["x"], s["res"] = normal(T, d), normal(T, d)
        s["router"] = normal(E, d, scale=d ** -0.5, kind=torch.float32)
        s["w13"], s["w2"] = normal(E, 2 * inter, d, scale=d ** -0.5), normal(E, d, inter, scale=inter ** -0.5)
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, part, layout):
    a, b = (x[..., :part // 2], x[..., part // 2:part]) if layout == "half" else (x[..., 0:part:2], x[..., 1:part:2])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat((u, v), -1) if layout == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((turned, x[..., part:]), -1)


def _plain_rope(s):
    angle = s["positions"].double()[..., None, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["amplitude"]).float(), (angle.sin() * s["amplitude"]).float()
    turn = lambda x, sn: _rotate(x.detach().float(), cos, sn, s["part"], s["layout"]).to(x.dtype)  # noqa: E731
    out = [turn(s["q"], sin), turn(s["k"], sin)]
    return out + [turn(s["dq"], -sin), turn(s["dk"], -sin)] if s["grad"] else out


def _act(z, act):
    """act(z) and its derivative."""
    one = torch.ones_like(z)
    if act == "none":
        return z, one
    if act == "relu":
        return z * (z > 0), one * (z > 0)
    if act == "leaky":
        slope = torch.where(z > 0, one, 0.01 * one)
        return z * slope, slope
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return z * g, g * (1 + z * (1 - g))
    if act == "tanh":
        th = torch.tanh(z)
        return th, 1 - th * th
    if act == "gelu_erf":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    t = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    h, slope = _act(x @ w.T + b, s["act"])
    y = (h if s["res"] is None else h + s["res"].detach().float()).to(t)
    if not s["grad"]:
        return [y]
    dz = s["dy"].float() * slope
    out = [y, (dz @ w).to(t), (dz.T @ x).to(t), dz.sum(0).to(t)]
    return out if s["res"] is None else out + [s["dy"]]


def _plain_moe(s):
    x = s["x"].float()
    p = torch.softmax(x @ s["router"].T, -1)
    top, chosen = (v[:, :s["top_k"]] for v in torch.sort(p, dim=-1, descending=True, stable=True))
    share = torch.zeros_like(p).scatter_(1, chosen, top / top.sum(-1, keepdim=True))
    gate, up = torch.matmul(x, s["w13"].float().transpose(1, 2)).chunk(2, -1)            # (E, T, inter): every expert on every token
    y = torch.matmul(gate / (1 + torch.exp(-gate)) * up, s["w2"].float().transpose(1, 2))
    y = s["res"].float() + (share.T[..., None] * y).sum(0)
    return [y.to(s["x"].dtype)]


# ---------------------------------------------------------------------------------------------------------------- the library's calls
def _own_rope(s):
    from autodiffusion_amd import ops, train
    if not s["grad"]:
        return list(ops.rope(s["q"], s["k"], s["positions"], s["inv_freq"], amplitude=s["amplitude"], layout=s["layout"]))
    q, k = train.rope(s["q"], s["k"], s["positions"], s["inv_freq"], amplitude=s["amplitude"], layout=s["layout"])
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]


def _own_linear(s):
    from autodiffusion_amd import ops, train
    act = ACTS.index(s["act"])
    if not s["grad"]:
        return [ops.linear_residual(s["x"], s["w"], s["b"], s["res"], act=act)]
    y = train.linear_residual(s["x"], s["w"], s["b"], s["res"], act=act)
    leaves = [v for v in (s["x"], s["w"], s["b"], s["res"]) if v is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def _own_moe(s):
    from autodiffusion_amd import str_backbone
    return [str_backbone.moe_few(s["x"], s["res"], s["router"], s["w13"], s["w2"], s["inter"], s["experts"], s["top_k"], PRECISION[s["type"]])]


PLAIN = {"rope": _plain_rope, "linear": _plain_linear, "moe": _plain_moe}
OWN = {"rope": _own_rope, "linear": _own_linear, "moe": _own_moe}


def run(state):
    return (OWN if own else PLAIN)[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- costs and exact values
def work(case):
    z = SIZE[case["type"]]
    if case["op"] == "rope":
        values = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["width"] * (2 if case["grad"] else 1)
        return {"bytes": 2 * values * z + 8 * case["batch"] * case["seq"], "flops": 3 * values * case["part"] // case["width"]}
    if case["op"] == "linear":
        M, N, K = case["rows"], case["n"], case["k"]
        forward = (M * K + N * K + N + M * N * (2 if case["residual"] else 1)) * z
        if not case["grad"]:
            return {"bytes": forward, "flops": 2 * M * N * K}
        return {"bytes": forward + (M * N + M * K + N * K + N) * z, "flops": 6 * M * N * K}
    T, d, inter, E, k = (case[n] for n in ("tokens", "d", "inter", "experts", "top_k"))
    experts = E * (1 - (1 - k / E) ** T)                   # expected number of distinct experts that T tokens choose
    return {"bytes": experts * 3 * d * inter * z + 4 * E * d + 3 * T * d * z, "flops": 6 * T * k * d * inter + 2 * T * E * d}


def _exact_rope(s):
    p, w, part = s["positions"].double(), s["inv_freq"], s["part"]
    turn = torch.polar(torch.full_like(w, s["amplitude"]).expand(*p.shape, part // 2).contiguous(), p.unsqueeze(-1) * w).unsqueeze(-2)

    def apply(x, by):
        x = x.detach().double()
        y = x.clone()
        first, second = (slice(0, part // 2), slice(part // 2, part)) if s["layout"] == "half" else (slice(0, part, 2), slice(1, part, 2))
        c = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        y[..., first], y[..., second] = c.real, c.imag
        return y

    out = [apply(s["q"], turn), apply(s["k"], turn)]
    return out + [apply(s["dq"], turn.conj()), apply(s["dk"], turn.conj())] if s["grad"] else out


def _exact_linear(s):
    d = {n: (None if s[n] is None else s[n].detach().double()) for n in ("x", "w", "b", "res")}
    d["x"], d["w"] = (v.requires_grad_() for v in (d["x"], d["w"]))
    f = torch.nn.functional
    act = {"none": lambda v: v, "relu": f.relu, "gelu_erf": f.gelu, "gelu_tanh": lambda v: f.gelu(v, approximate="tanh"),
           "leaky": lambda v: f.leaky_relu(v, 0.01), "silu": f.silu, "tanh": torch.tanh}[s["act"]]
    with torch.enable_grad():
        b = d["b"].requires_grad_()
        y = act(torch.addmm(b, d["x"], d["w"].t()))
        if d["res"] is not None:
            y = y + d["res"]
    if not s["grad"]:
        return [y.detach()]
    out = [y.detach(), *torch.autograd.grad(y, (d["x"], d["w"], b), s["dy"].double())]
    return out if d["res"] is None else out + [s["dy"].double()]


def _exact_moe(s):
    x = s["x"].double()
    logits = torch.einsum("td,ed->te", x, s["router"].double())
    y = s["res"].double()
    chosen = logits.topk(s["top_k"], dim=-1).indices
    kept = torch.full_like(logits, -math.inf).scatter(1, chosen, logits.gather(1, chosen))
    share = torch.softmax(kept, -1)                        # over the chosen ones alone: the renormalised probabilities
    for e in range(s["experts"]):
        rows = (share[:, e] > 0).nonzero()[:, 0]
        if len(rows):
            g, u = (x[rows] @ s["w13"][e].double().t()).split(s["inter"], dim=1)
            y[rows] += share[rows, e, None] * ((g * torch.sigmoid(g) * u) @ s["w2"][e].double().t())
    return [y]


def exact(case, seed):
    return {"rope": _exact_rope, "linear": _exact_linear, "moe": _exact_moe}[case["op"]](prepare(case, seed))
