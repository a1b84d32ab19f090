"""Workloads of the training operators that stand beside the network kernels: group normalisation with an activation
over channels-last data (forward, and forward + backward), the orthogonalised form of a matrix by Newton-Schulz products,
and a Muon step over the hidden matrices of a network.

`run` computes each in elementary torch operations, or (`own`) through dex_gan_grasp_amd.  Shapes follow the networks of
this repository: hidden rows of 256 / 512 units, fused fc1 || fc3 rows of 768, point clouds of 2048 points, fc matrices of
256 / 512 rows and 4101 .. 4620 columns, heads of 12 rows.
"""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)   # quintic x -> a x + b x^3 + c x^5 of the Newton-Schulz iteration
STEPS = 5
NS_EPS = 1e-7
GN_EPS = 1e-5
SLOPE = 0.2                         # LeakyReLU of the ResBlocks
LR, MU, WD = 0.02, 0.95, 0.01
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one small inference batch of hidden rows: launch latency
        dict(name="gn rows 32 f32 fwd", op="gn", mode="fwd", n=32, s=1, c=512, g=32, pitch=512, act="leaky_relu", dtype="f32"),
        # a train step's batch: the 512 fc3 columns inside the fused 768-column product, one group of 16 units each
        dict(name="gn rows 1024 f32 train", op="gn", mode="train", n=1024, s=1, c=512, g=32, pitch=768, act="leaky_relu",
             dtype="f32"),
        # per-point features of odd-sized clouds, 12 channels to a group
        dict(name="gn odd clouds f16 train", op="gn", mode="train", n=5, s=1237, c=132, g=11, pitch=132, act="silu",
             dtype="f16"),
        # per-point features of a batch of 2048-point clouds in training
        dict(name="gn clouds bf16 train", op="gn", mode="train", n=32, s=2048, c=256, g=32, pitch=256, act="leaky_relu",
             dtype="bf16"),
        # the same for a large inference batch
        dict(name="gn clouds bf16 fwd", op="gn", mode="fwd", n=128, s=2048, c=256, g=32, pitch=256, act="silu", dtype="bf16"),
        # one output head (12 joints x 512 units): latency
        dict(name="ns head f32", op="ns", count=1, rows=12, cols=512, dtype="f32"),
        # one fc2 matrix, taller than wide
        dict(name="ns fc2 f32", op="ns", count=1, rows=512, cols=256, dtype="f32"),
        # a stack of odd-sized matrices
        dict(name="ns stack f32", op="ns", count=24, rows=257, cols=771, dtype="f32"),
        # the widest fc3 matrix with a bf16 gradient
        dict(name="ns fc3 bf16", op="ns", count=1, rows=512, cols=4620, dtype="bf16"),
        # optimiser step of a one-block toy network: latency
        dict(name="muon toy", op="muon", fin=77, blocks=1, hidden=32, out=64),
        # the generator's hidden matrices
        dict(name="muon generator", op="muon", fin=4101, blocks=2, hidden=256, out=512),
        # the evaluator's hidden matrices
        dict(name="muon evaluator", op="muon", fin=4108, blocks=3, hidden=256, out=512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gn", "gn", "ns", "muon"))
    if op == "gn":
        mode = rng.choice(("fwd", "train"))
        d = _log(rng, 1, 64)
        g = _log(rng, 1, max(1, min(64, 1024 // d)))
        c = d * g
        most = (1 << 26 if mode == "fwd" else 1 << 24) // c        # rows that the largest listed case of the mode allows
        s = 1 if rng.random() < 0.3 else _log(rng, 1, min(most, 70000))
        n = _log(rng, 1, max(1, min(most // s, 4096)))
        pitch = c + (rng.randint(1, 64) if rng.random() < 0.3 else 0)
        return dict(op="gn", mode=mode, n=n, s=s, c=c, g=g, pitch=pitch, act=rng.choice(("leaky_relu", "silu", "none")),
                    dtype=rng.choice(("f32", "bf16", "f16")))
    if op == "ns":
        small = _log(rng, 1, 512)
        large = _log(rng, small, 4620)
        rows, cols = (small, large) if rng.random() < 0.7 else (large, small)
        count = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, min(32, 6 * 512 * 512 * 4620 // (small * small * large))))
        return dict(op="ns", count=count, rows=rows, cols=cols, dtype=rng.choice(("f32", "bf16", "f16")))
    return dict(op="muon", fin=_log(rng, 16, 4108), blocks=rng.randint(1, 3), hidden=_log(rng, 16, 256),
                out=_log(rng, 16, 512))


def _shapes(case):
    """The hidden matrices of a stack of ResBlocks: fc1 (hidden, f), fc3 (out, f), fc2 (out, hidden) for each block, whose
    input f is the network's input and, behind the first block, the previous block's output as well."""
    for b in range(case["blocks"]):
        f = case["fin"] + (case["out"] if b else 0)
        yield case["hidden"], f
        yield case["out"], f
        yield case["out"], case["hidden"]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _gradient(gen, rows, cols, count=1):
    """What a weight gradient is: dy^T x over a batch, the units' scales spread over a decade, divided by the batch."""
    b = 1024
    dy = _randn(gen, count, b, rows) * torch.logspace(0, -1, rows, device="cuda")
    x = _randn(gen, count, b, cols) * torch.logspace(0, -0.5, cols, device="cuda")
    return (dy.transpose(1, 2).contiguous() @ x) / b


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    state = dict(case)
    if case["op"] == "gn":
        n, s, c, dt = case["n"], case["s"], case["c"], DTYPES[case["dtype"]]
        # pre-activations with a mean and a scale of their own in every channel
        rows = torch.empty((n, s, case["pitch"]), device="cuda", dtype=dt)
        rows.normal_(generator=gen)
        x = rows[:, :, case["pitch"] - c:]
        x.mul_((0.5 + torch.rand(c, generator=gen, device="cuda")).to(dt)).add_((0.3 * _randn(gen, c)).to(dt))
        state.update(x=x, weight=1.0 + 0.1 * _randn(gen, c), bias=0.1 * _randn(gen, c))
        if case["mode"] == "train":
            dy = torch.empty((n, s, c), device="cuda", dtype=dt)
            state["dy"] = dy.normal_(generator=gen)
    elif case["op"] == "ns":
        g = _gradient(gen, case["rows"], case["cols"], case["count"]).to(DTYPES[case["dtype"]])
        state["grad"] = g if case["count"] > 1 else g[0]
    else:
        shapes = list(_shapes(case))
        state["grads"] = [_gradient(gen, r, c)[0] for r, c in shapes]
        state["momentum"] = [8.0 * _gradient(gen, r, c)[0] for r, c in shapes]   # of the steps before
        state["params"] = [_randn(gen, r, c) / math.sqrt(c) for r, c in shapes]
    return state


def _group_norm(st):
    """y = act(weight * (x - mean) / sqrt(var + eps) + bias), mean and var over the points and channels of a group; the
    gradients by the formulas of the backward pass.  LeakyReLU's statistics and pre-activations in 64 bits: which side of
    the kink an element lies on decides its gradient."""
    n, s, c, g = st["n"], st["s"], st["c"], st["g"]
    wide = torch.float64 if st["act"] == "leaky_relu" else torch.float32
    dt = st["x"].dtype
    x = st["x"].to(wide).reshape(n, s, g, c // g)
    mean = x.mean(dim=(1, 3), keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(dim=(1, 3), keepdim=True) + GN_EPS)
    xhat = xc * rstd
    w, b = st["weight"].to(wide).view(g, c // g), st["bias"].to(wide).view(g, c // g)
    z = xhat * w + b
    if st["act"] == "leaky_relu":
        y, slope = torch.where(z > 0, z, SLOPE * z), torch.where(z > 0, 1.0, SLOPE)
    elif st["act"] == "silu":
        sig = torch.sigmoid(z)
        y, slope = z * sig, sig * (1.0 + z * (1.0 - sig))
    else:
        y, slope = z, torch.ones_like(z)
    y = y.reshape(n, s, c).to(dt)
    if st["mode"] == "fwd":
        return y
    dz = st["dy"].to(wide).reshape(n, s, g, c // g) * slope
    dxh = dz * w
    dx = rstd * (dxh - dxh.mean(dim=(1, 3), keepdim=True) - xhat * (dxh * xhat).mean(dim=(1, 3), keepdim=True))
    dweight, dbias = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    return {"y": y, "dx": dx.reshape(n, s, c).to(dt), "dweight": dweight.reshape(c).float(), "dbias": dbias.reshape(c).float()}


def _newton_schulz(g):
    """X_0 = g / (|g| + eps); X <- a X + (b A + c A^2) X with A = X X^T over the shorter side."""
    x = g.float()
    turned = x.shape[-2] > x.shape[-1]
    if turned:
        x = x.transpose(-1, -2).contiguous()
    a, b, c = COEF
    x = x / (torch.sqrt((x * x).sum(dim=(-1, -2), keepdim=True)) + NS_EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if turned else x


def run(state):
    if own:
        from dex_gan_grasp_amd import ops
        if state["op"] == "gn":
            args = (state["x"], state["g"], state["weight"], state["bias"], GN_EPS, state["act"], SLOPE)
            if state["mode"] == "fwd":
                return ops.group_norm_act_forward(*args)[0]
            y, stats = ops.group_norm_act_forward(*args)
            dx, dweight, dbias = ops.group_norm_act_backward(state["dy"], *args, stats)
            return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
        if state["op"] == "ns":
            return ops.orthogonalize(state["grad"], STEPS, COEF, NS_EPS)
        ops.muon_step(state["params"], state["grads"], state["momentum"], LR, MU, True, WD, STEPS, COEF, NS_EPS)
        return {"params": state["params"], "momentum": state["momentum"]}
    if state["op"] == "gn":
        return _group_norm(state)
    if state["op"] == "ns":
        return _newton_schulz(state["grad"]).to(state["grad"].dtype)
    for w, g, m in zip(state["params"], state["grads"], state["momentum"]):
        m.mul_(MU).add_(g)
        o = _newton_schulz(g + MU * m)
        w.mul_(1.0 - LR * WD).sub_(o, alpha=LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1])))
    return {"params": state["params"], "momentum": state["momentum"]}


def _ns_work(rows, cols):
    """A and A^2 are symmetric: half of their entries are enough."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def work(case):
    if case["op"] == "gn":
        e, size = case["n"] * case["s"] * case["c"], DTYPES[case["dtype"]].itemsize
        passes, flops = (2, 8) if case["mode"] == "fwd" else (4, 24)      # x, y; and dy, dx
        return {"bytes": passes * e * size + (4 if passes == 4 else 2) * case["c"] * 4, "flops": flops * e}
    if case["op"] == "ns":
        e = case["count"] * case["rows"] * case["cols"]
        return {"bytes": 2 * e * DTYPES[case["dtype"]].itemsize, "flops": case["count"] * _ns_work(case["rows"], case["cols"])}
    # parameters, gradients and momentum read, parameters and momentum written
    return {"bytes": sum(20 * r * c for r, c in _shapes(case)), "flops": sum(_ns_work(r, c) for r, c in _shapes(case))}


def _exact_gn(st):
    n, s, c, g = st["n"], st["s"], st["c"], st["g"]
    d = c // g
    size = s * d
    x = st["x"].double().reshape(n, s, g, d).permute(0, 2, 1, 3).reshape(n * g, size)      # one row a group
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    inv = (var + GN_EPS) ** -0.5
    w = st["weight"].double().view(1, g, 1, d).expand(n, g, s, d).reshape(n * g, size)
    b = st["bias"].double().view(1, g, 1, d).expand(n, g, s, d).reshape(n * g, size)
    h = (x - mean) * inv
    z = w * h + b
    back = lambda v: v.view(n, g, s, d).permute(0, 2, 1, 3).reshape(n, s, c)   # noqa: E731
    if st["act"] == "leaky_relu":
        pos = (z > 0).double()
        y, dact = z * (pos + SLOPE * (1 - pos)), pos + SLOPE * (1 - pos)
    elif st["act"] == "silu":
        e = 1.0 / (1.0 + torch.exp(-z))
        y, dact = z * e, e + z * e * (1 - e)
    else:
        y, dact = z, torch.ones_like(z)
    if st["mode"] == "fwd":
        return back(y)
    gz = st["dy"].double().reshape(n, s, g, d).permute(0, 2, 1, 3).reshape(n * g, size) * dact
    gh = gz * w
    dx = inv / size * (size * gh - gh.sum(1, keepdim=True) - h * (gh * h).sum(1, keepdim=True))
    return {"y": back(y), "dx": back(dx), "dweight": back(gz * h).sum((0, 1)), "dbias": back(gz).sum((0, 1))}


def _exact_orthogonal(g):
    """The polynomial of the singular values: U p(...p(s / |g|)) V^T, without a decomposition, as a product by the shorter
    side's Gram matrix in every step."""
    g = g.double()
    if g.shape[-2] > g.shape[-1]:
        return _exact_orthogonal(g.transpose(-1, -2)).transpose(-1, -2)
    x = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + NS_EPS)
    one = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.mT.contiguous())
        x = torch.matmul(COEF[0] * one + torch.matmul(gram, COEF[1] * one + COEF[2] * gram), x)
    return x


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "gn":
        return _exact_gn(st)
    if case["op"] == "ns":
        return _exact_orthogonal(st["grad"])
    out = {"params": [], "momentum": []}
    for w, g, m in zip(st["params"], st["grads"], st["momentum"]):
        m = MU * m.double() + g.double()
        o = _exact_orthogonal(g.double() + MU * m)
        out["params"].append((1.0 - LR * WD) * w.double() - LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * o)
        out["momentum"].append(m)
    return out
