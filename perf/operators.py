"""Cases by which the training-step operators are timed: layer normalisation (forward, and forward + backward with the
sums of the weight gradients), Newton-Schulz orthogonalisation of a gradient, and the Muon update built on it.

`own = False` computes every operator in its plain form (elementary tensor operations in fp32); `own = True` makes the
calls a training program makes of `gan_flow_amd`."""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # Muon's quintic
STEPS, NS_EPS, LN_EPS = 5, 1e-7, 1e-5
LR, MOMENTUM, WEIGHT_DECAY = 1e-3, 0.95, 0.1
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one small evaluation batch through a hidden layer of the wide (256) nets: latency of one launch
        dict(name="norm_16x256_fp32", op="norm", rows=16, cols=256, dtype="fp32", wdtype="fp32", pad=0, train=False),
        # a large inference batch of activations in bf16: bandwidth
        dict(name="norm_16384x4096_bf16", op="norm", rows=16384, cols=4096, dtype="bf16", wdtype="bf16", pad=0, train=False),
        # the training batch (2 048 rows) at hidden width 256, forward and backward
        dict(name="norm_train_2048x256_fp32", op="norm", rows=2048, cols=256, dtype="fp32", wdtype="fp32", pad=0, train=True),
        # odd sizes, rows that are slices of a wider buffer, fp32 weights beside fp16 activations
        dict(name="norm_train_4099x1001_fp16", op="norm", rows=4099, cols=1001, dtype="fp16", wdtype="fp32", pad=30, train=True),
        # a long training batch in bf16: bandwidth of both directions
        dict(name="norm_train_32768x2048_bf16", op="norm", rows=32768, cols=2048, dtype="bf16", wdtype="bf16", pad=0, train=True),
        # one hidden matrix of the 64-wide ODE net
        dict(name="orth_1x64x64_fp32", op="orth", count=1, rows=64, cols=64, dtype="fp32"),
        # the hidden matrices of four blocks of the 256-wide ODE net
        dict(name="orth_8x256x256_fp32", op="orth", count=8, rows=256, cols=256, dtype="fp32"),
        # a tall matrix of odd sizes in bf16
        dict(name="orth_1x1000x333_bf16", op="orth", count=1, rows=1000, cols=333, dtype="bf16"),
        # the largest square matrix
        dict(name="orth_1x4096x4096_bf16", op="orth", count=1, rows=4096, cols=4096, dtype="bf16"),
        # the optimizer step of the 64-wide ODE net's two hidden matrices
        dict(name="muon_2x64x64_fp32", op="muon", count=2, rows=64, cols=64, dtype="fp32"),
        # the tall input projections of a layer stack, bf16 weights
        dict(name="muon_8x1024x512_bf16", op="muon", count=8, rows=1024, cols=512, dtype="bf16"),
        # the wide projections of a layer stack, fp32 weights
        dict(name="muon_4x1024x4096_fp32", op="muon", count=4, rows=1024, cols=4096, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _products(case):
    m, n = sorted((case["rows"], case["cols"]))
    return case["count"] * STEPS * (3 * m * m * n + m * m * m)


def draw(rng):
    op = rng.choice(["norm", "norm", "orth", "muon"])
    if op == "norm":
        cols = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(32768, (1 << 26) // cols))
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        return dict(op="norm", rows=rows, cols=cols, dtype=dtype, wdtype=rng.choice([dtype, "fp32"]), pad=rng.choice([0, 0, 1, 24]),
                    train=rng.random() < 0.7)
    dtype = rng.choice(["fp32", "bf16", "fp16"] if op == "orth" else ["fp32", "bf16"])
    case = dict(op=op, count=_log_int(rng, 1, 16), rows=_log_int(rng, 24, 2048), cols=_log_int(rng, 24, 4096), dtype=dtype)
    if rng.random() < 0.5:
        case["rows"], case["cols"] = case["cols"], case["rows"]
    while case["count"] > 1 and _products(case) > STEPS * 4 * 4096 ** 3 // 8:
        case["count"] -= 1
    return case


def _gradient(count, rows, cols, g, dev):
    """What a layer's gradient looks like: a decaying spectrum over a floor of noise, at a gradient's scale."""
    r = min(rows, cols)
    decay = torch.logspace(0, -3, r, device=dev)
    u = torch.randn(count, rows, r, generator=g, device=dev)
    v = torch.randn(count, r, cols, generator=g, device=dev)
    noise = torch.randn(count, rows, cols, generator=g, device=dev)
    return 1e-3 * ((u * decay) @ v / math.sqrt(r) + 0.1 * noise)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, cols, wdt = case["rows"], case["cols"], DTYPES[case["wdtype"]]

        def activations(shift):
            wide = torch.randn(rows, cols + case["pad"], generator=g, device=dev)
            wide[:, ::97] *= 8.0                                     # a few loud features, as activations have them
            return (wide + shift).to(dt)[:, :cols]

        x, dy = activations(torch.randn(rows, 1, generator=g, device=dev)), activations(0.0)
        w = (1.0 + 0.2 * torch.randn(cols, generator=g, device=dev)).to(wdt)
        b = (0.2 * torch.randn(cols, generator=g, device=dev)).to(wdt)
        if case["train"]:
            for t in (x, w, b):
                t.requires_grad_(True)
        return dict(case=case, x=x, dy=dy, w=w, b=b)
    grad = _gradient(case["count"], case["rows"], case["cols"], g, dev).to(dt)
    if case["op"] == "orth":
        return dict(case=case, g=grad)
    fan = math.sqrt(case["cols"])
    w = (torch.randn(grad.shape, generator=g, device=dev) / fan).to(dt)
    buf = 3.0 * _gradient(case["count"], case["rows"], case["cols"], g, dev)   # the momentum some steps into a training
    return dict(case=case, g=grad, w=w, m=buf, lists=[list(t.unbind(0)) for t in (w, grad, buf)])


def _plain_norm(x, w, b):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    c = xf - mean
    rstd = (c.square().mean(-1, keepdim=True) + LN_EPS).rsqrt()
    return (c * rstd * w.float() + b.float()).to(x.dtype)


def _plain_orthogonalize(g):
    """fp32 in, fp32 out; the smaller side on the left."""
    a, b, c = COEFFICIENTS
    tall = g.shape[-2] > g.shape[-1]
    x = (g.transpose(-2, -1) if tall else g).contiguous()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS).float()
    for _ in range(STEPS):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.transpose(-2, -1) if tall else x


def _scale(rows, cols):
    return 0.2 * math.sqrt(max(rows, cols))


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        x, w, b = state["x"], state["w"], state["b"]
        if own:
            from gan_flow_amd.lib.layers import layer_norm
            y = layer_norm(x, w, b, LN_EPS)
        else:
            y = _plain_norm(x, w, b)
        if not case["train"]:
            return [y]
        return [y.detach()] + list(torch.autograd.grad(y, (x, w, b), state["dy"]))
    if case["op"] == "orth":
        if own:
            from gan_flow_amd.lib.optim import orthogonalize
            return [orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)]
        return [_plain_orthogonalize(state["g"].float()).to(state["g"].dtype).contiguous()]
    w, g, m = state["w"], state["g"], state["m"]
    if own:
        from gan_flow_amd.lib.optim import muon_step
        params, grads, momenta = state["lists"]
        muon_step(params, grads, momenta, lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=WEIGHT_DECAY,
                  scale=_scale(case["rows"], case["cols"]), steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    else:
        gf = g.float()
        m.mul_(MOMENTUM).add_(gf)
        o = _plain_orthogonalize(gf + MOMENTUM * m)
        w.copy_(w.float() * (1.0 - LR * WEIGHT_DECAY) - (LR * _scale(case["rows"], case["cols"])) * o)
    return [w, m]


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "norm":
        n, e, we = case["rows"] * case["cols"], size[case["dtype"]], size[case["wdtype"]]
        if not case["train"]:
            return dict(bytes=2 * n * e + 2 * case["cols"] * we, flops=8 * n)
        return dict(bytes=5 * n * e + 5 * case["cols"] * we, flops=22 * n)   # x, y; x, dy, dx; w, b; w, dw, db
    n, e = case["count"] * case["rows"] * case["cols"], size[case["dtype"]]
    # per step: the Gram matrix and its square are symmetric (half of their products), the last product is full
    return dict(bytes=2 * n * e if case["op"] == "orth" else 3 * n * e + 8 * n, flops=_products(case))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b, dy = (state[k].detach().double() for k in ("x", "w", "b", "dy"))
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        inv = 1.0 / torch.sqrt(var + LN_EPS)
        xh = (x - mean) * inv
        y = xh * w + b
        if not case["train"]:
            return [y]
        h = dy * w
        dx = inv * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
        return [y, dx, (dy * xh).sum(0), dy.sum(0)]

    def polynomial(u):
        # the same polynomial of the singular values from the other side: the smaller Gram matrix, multiplied on the right
        a, b, c = COEFFICIENTS
        wide = u.shape[2] > u.shape[1]
        t = u.transpose(1, 2).contiguous() if wide else u
        t = t / (torch.linalg.vector_norm(t, dim=(1, 2), keepdim=True) + NS_EPS)
        eye = torch.eye(t.shape[2], dtype=t.dtype, device=t.device)
        for _ in range(STEPS):
            r = torch.matmul(t.transpose(1, 2).contiguous(), t)
            t = torch.matmul(t, a * eye + b * r + c * torch.matmul(r, r))
        return t.transpose(1, 2) if wide else t

    g = state["g"].double()
    if case["op"] == "orth":
        return [polynomial(g).contiguous()]
    m = MOMENTUM * state["m"].double() + g
    o = polynomial(g + MOMENTUM * m)
    return [state["w"].double() * (1.0 - LR * WEIGHT_DECAY) - LR * _scale(case["rows"], case["cols"]) * o, m]
