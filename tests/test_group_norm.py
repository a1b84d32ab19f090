"""Group normalisation with an activation over channels-last data (ops.group_norm_act_forward / _backward) against its formulas in
64 bits on the CPU, at the sizes, strides and values where it can go wrong, and its refusals.

Tolerances.  Statistics, xh and z are 64-bit inside, so an element's side of LeakyReLU's kink is the reference's; what follows is
fp32 (unit roundoff u = 2^-24) and one rounding to the output type (half a step, eps/2; 2^-25 absolute where float16 is subnormal):
  y : z rounded (u), times slope (u) or / (1 + exp(-z)): exp of a rounded argument is off by |z| u + 2u, the sum and the quotient
      by u each                                                   -> (eps/2 + (8 + |z|) u) |y|
  dx: each of w dz, mean(w dz), xh mean(w dz xh) is rounded and multiplied by a rounded factor; SiLU's slope carries (8 + |z|) u of
      |dy| (1 + |z|) -> eps/2 |dx| + u rstd (8 + |z|)(...) summed below
  dw, db: 64-bit sums of terms off by (8 + |z|) u each, partial sums stored in fp32 (u) -> u sum((10 + |z|) |term|)"""
import itertools

import pytest
import torch

from dex_gan_grasp_amd import _lib, ops

U = 2.0 ** -24


def reference(x, dy, groups, w, b, eps, act, slope):
    """The formulas on CPU doubles; dict of y, dx, dw, db and of what the tolerances are made of."""
    n, c = x.shape[0], x.shape[-1]
    x = x.double().reshape(n, -1, groups, c // groups)
    w = (torch.ones(c) if w is None else w).double().view(groups, -1)
    b = (torch.zeros(c) if b is None else b).double().view(groups, -1)
    mean = x.mean((1, 3), keepdim=True)
    rstd = (((x - mean) ** 2).mean((1, 3), keepdim=True) + eps) ** -0.5
    xh = (x - mean) * rstd
    z = xh * w + b
    if act == "leaky_relu":
        d = torch.where(z > 0, 1.0, slope).double()
        y = z * d
    elif act == "silu":
        s = torch.sigmoid(z)
        y, d = z * s, s * (1 + z * (1 - s))
    else:
        y, d = z, torch.ones_like(z)
    dy = dy.double().reshape(x.shape)
    dz = dy * d
    wd = dz * w
    m1, m2 = wd.mean((1, 3), keepdim=True), (wd * xh).mean((1, 3), keepdim=True)
    dx = rstd * (wd - m1 - xh * m2)
    unsure = (8 + z.abs()) * U * dy.abs() * (d.abs() + (1 + z.abs() if act == "silu" else 0))   # of dz
    wu = unsure * w.abs()
    dx_tol = rstd * (wu + wu.mean((1, 3), keepdim=True) + xh.abs() * (wu * xh.abs()).mean((1, 3), keepdim=True)
                     + 6 * U * (wd.abs() + m1.abs() + xh.abs() * m2.abs()))
    return dict(y=y, z=z, dx=dx, dx_tol=dx_tol, mean=mean, rstd=rstd, dw=(dz * xh).sum((0, 1)).reshape(-1),
                db=dz.sum((0, 1)).reshape(-1), dw_tol=((unsure + 2 * U * dz.abs()) * xh.abs()).sum((0, 1)).reshape(-1),
                db_tol=(unsure + 2 * U * dz.abs()).sum((0, 1)).reshape(-1))


def half_step(dtype, ref):
    return torch.finfo(dtype).eps / 2 * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def close(got, ref, tol, what):
    bad = (got.double().cpu().reshape(ref.shape) - ref).abs() > tol
    assert not bad.any(), "%s: %d of %d outside, worst off by %.3g (allowed %.3g)" % (
        what, int(bad.sum()), bad.numel(), float((got.double().cpu().reshape(ref.shape) - ref).abs()[bad].max()), float(tol[bad].min()))


def check(x, dy, groups, w, b, eps=1e-5, act="leaky_relu", slope=0.2, dev="cuda"):
    """x, dy: CPU tensors or (their device versions with strides of their own)."""
    xd, dyd = (t if t.is_cuda else t.to(dev) for t in (x, dy))
    wd, bd = (None if t is None else t.to(dev) for t in (w, b))
    y, stats = ops.group_norm_act_forward(xd, groups, wd, bd, eps, act, slope)
    dx, dw, db = ops.group_norm_act_backward(dyd, xd, groups, wd, bd, eps, act, slope, stats)
    r = reference(x.cpu(), dy.cpu(), groups, w, b, eps, act, slope)
    dt = x.dtype
    assert y.dtype == dx.dtype == dt and y.shape == dx.shape == x.shape and y.is_contiguous() and dx.is_contiguous()
    close(stats[..., 1], r["rstd"].reshape(stats.shape[:2]), 1e-12 * r["rstd"].reshape(stats.shape[:2]), "rstd")
    close(y, r["y"], half_step(dt, r["y"]) + (8 + r["z"].abs()) * U * r["y"].abs(), "y")
    close(dx, r["dx"], half_step(dt, r["dx"]) + r["dx_tol"], "dx")
    close(dw, r["dw"], r["dw_tol"] + U * r["dw"].abs(), "dweight")
    close(db, r["db"], r["db_tol"] + U * r["db"].abs(), "dbias")
    return y, dx, dw, db


def data(shape, dtype, seed, scale=1.0, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * scale * (0.5 + torch.rand(c, generator=g)) + shift * torch.randn(c, generator=g)).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    return x, dy, 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)


# (N, S, C, groups): one point, one channel a group, groups of 3 / 12 / 16 / 2048 channels, rows, short and long samples, sizes on
# both sides of every route's limit, more samples than workgroups
SHAPES = [(1, 1, 1, 1), (1, 1, 512, 32), (3, 1, 6, 6), (2, 1, 2048, 1), (2, 1, 4096, 1), (2, 1, 4100, 1), (2, 1, 513, 1), (7, 1, 515, 1),
          (33, 1, 768, 48), (1030, 1, 96, 8), (5, 1, 12, 3), (4, 2, 512, 32), (2, 64, 32, 4), (2, 65, 32, 1), (3, 37, 132, 11),
          (2, 300, 8, 8), (1, 5000, 24, 2), (2, 129, 1030, 5), (1, 70, 2100, 3), (300, 3, 20, 5), (2, 1000, 3, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_matches_formulas(shape, dtype):
    n, s, c, g = shape
    for act in ("leaky_relu", "silu", "none"):
        x, dy, w, b = data((n, s, c), dtype, n + s + c + g)
        check(x, dy, g, w, b, act=act)
    check(x, dy, g, None, None, eps=0.1, act="leaky_relu", slope=0.0)


@pytest.mark.gpu
def test_two_and_four_dimensional_inputs_and_no_parameter_gradients():
    x, dy, w, b = data((6, 64), torch.float32, 1)
    check(x, dy, 4, w, b)
    x, dy, w, b = data((2, 5, 7, 24), torch.bfloat16, 2)
    check(x, dy, 4, w, b)
    xd, dyd, wd, bd = (t.cuda() for t in (x, dy, w, b))
    y, st = ops.group_norm_act_forward(xd, 4, wd, bd)
    dx, dw, db = ops.group_norm_act_backward(dyd, xd, 4, wd, bd, 1e-5, "leaky_relu", 0.2, st, param_grads=False)
    full = ops.group_norm_act_backward(dyd, xd, 4, wd, bd, 1e-5, "leaky_relu", 0.2, st)
    assert dw is None and db is None and torch.equal(dx, full[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape", [(40, 1, 512, 32), (3, 70, 512, 32)], ids=["rows", "points"])
def test_strides_and_alignment(shape, dtype):
    n, s, c, g = shape
    x, dy, w, b = data((n, s, c), dtype, 3)
    want = [t.clone() for t in check(x, dy, g, w, b)]
    wide = torch.full((n, s, 768 + 8), 7.0, dtype=dtype, device="cuda")
    for off in (256, 257, 260):                       # a column block of a wider product: aligned, odd, half-way
        wide[:, :, off:off + c] = x.cuda()
        check(wide[:, :, off:off + c], dy, g, w, b)
    order = x.cuda().permute(1, 2, 0).contiguous().permute(2, 0, 1)     # channels not side by side: copied
    got = check(order, dy.cuda().transpose(0, 1).contiguous().transpose(0, 1), g, w, b)
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    one = dy[:1, :1].cuda().expand(n, s, c)           # a broadcast gradient, as a sum's backward hands down
    check(x, one, g, w, b)
    flat = torch.zeros(n * s * c + 3, dtype=dtype, device="cuda")       # a base that is not 16-byte aligned
    view = flat[3:].view(n, s, c)
    view.copy_(x)
    check(view, dy, g, w, b)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 1, 64, 4), (2, 700, 64, 4)], ids=["rows", "points"])
def test_values_where_it_can_go_wrong(shape):
    n, s, c, g = shape
    # far from zero: the variance is 1e-6 of the square of the mean
    x, dy, w, b = data((n, s, c), torch.float32, 5)
    check(x + 1000.0, dy, g, w, b)
    check(x * 1e-18, dy, g, w, b)                     # eps decides
    check(x * 1e18, dy, g, w, b, act="none")          # squares beyond fp32
    # a constant group: z is the bias exactly — at the kink itself without one (slope side, as z > 0 is false)
    const = torch.full((n, s, c), 0.1)
    y, dx, _, db = check(const, dy, g, None, None)
    assert not y.any()
    check(const, dy, g, w, b)
    # NaN and infinity stay inside their sample and group
    for bad in (float("nan"), float("inf")):
        xb = x.clone()
        xb[1, -1, 17] = bad
        xd = xb.cuda()
        y, st = ops.group_norm_act_forward(xd, g, w.cuda(), b.cuda())
        dx, dw, _ = ops.group_norm_act_backward(dy.cuda(), xd, g, w.cuda(), b.cuda(), 1e-5, "leaky_relu", 0.2, st)
        ok = torch.ones(n, s, c, dtype=torch.bool)
        ok[1, :, 16:32] = False
        for t, want in ((y, ops.group_norm_act_forward(x.cuda(), g, w.cuda(), b.cuda())[0]),):
            assert torch.equal(t.cpu()[ok], want.cpu()[ok]) and t.cpu()[~ok].isnan().all()
        assert dx.cpu()[~ok].isnan().all() and not dx.cpu()[ok].isnan().any()
        cols = torch.ones(c, dtype=torch.bool)
        cols[16:32] = False
        assert not dw.cpu()[cols].isnan().any() and dw.cpu()[~cols].isnan().all()


@pytest.mark.gpu
def test_empty_inputs():
    for shape in ((0, 8), (0, 3, 8), (2, 0, 8)):
        x = torch.zeros(shape, device="cuda")
        w = torch.ones(8, device="cuda")
        y, st = ops.group_norm_act_forward(x, 2, w, w)
        dx, dw, db = ops.group_norm_act_backward(x, x, 2, w, w, 1e-5, "silu", 0.2, st)
        assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "none"])
def test_gradients_against_differences(act):
    """Central differences of sum(y * dy) in the operator's own forward, at a step where fp32 outputs leave 1e-3 of the result."""
    x, dy, w, b = data((2, 3, 12), torch.float32, 9)
    xd, dyd, wd, bd = (t.cuda() for t in (x, dy, w, b))
    y, st = ops.group_norm_act_forward(xd, 3, wd, bd, 1e-5, act)
    dx, dw, db = ops.group_norm_act_backward(dyd, xd, 3, wd, bd, 1e-5, act, 0.2, st)
    f = lambda *t: float((ops.group_norm_act_forward(t[0], 3, t[1], t[2], 1e-5, act)[0].double() * dyd.double()).sum())   # noqa: E731
    h = 2.0 ** -7
    for k, grad in ((0, dx), (1, dw), (2, db)):
        for i in itertools.islice(range(grad.numel()), 0, None, 5):
            up, dn = ([t.clone() for t in (xd, wd, bd)] for _ in range(2))
            up[k].view(-1)[i] += h
            dn[k].view(-1)[i] -= h
            num = (f(*up) - f(*dn)) / (2 * h)
            # the third derivative's term h^2 / 6 stays below 1e-3 for these inputs of order one; 36 outputs rounded to fp32 are
            # off by 36 * 2^-24 * 4 / (2 h) < 6e-4
            assert abs(num - float(grad.view(-1)[i])) < 2e-3 * (1 + abs(num)), (k, i, num, float(grad.view(-1)[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(64, 1, 512, 32), (4, 300, 64, 8)], ids=["rows", "points"])
def test_other_streams_repeats_and_graph_replays(shape):
    n, s, c, g = shape
    x, dy, w, b = (t.cuda() for t in data((n, s, c), torch.float32, 11))
    args = (g, w, b, 1e-5, "leaky_relu", 0.2)

    def both():
        y, st = ops.group_norm_act_forward(x, *args)
        return (y,) + ops.group_norm_act_backward(dy, x, *args, st)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    for a, e in zip(got, want):
        assert torch.equal(a, e)        # no atomics: the same bits
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        x.copy_(data((n, s, c), torch.float32, 20 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, both()):
            assert torch.equal(a, e), k


def test_refusals_without_a_gpu():
    with pytest.raises(_lib.DggError):
        ops.group_norm_act_forward(torch.zeros(2, 8), 2)
    lib = _lib.lib()
    ws = lib.dgg_group_norm_workspace_bytes
    assert ws(32, 2048, 256, 32, _lib.BF16, 1) > 0 and ws(4, 100000, 8, 2, _lib.F32, 0) > 0 and ws(32, 1, 512, 32, _lib.F32, 0) >= 0
    for bad in ((0, 1, 8, 2, 0, 0), (1, 0, 8, 2, 0, 0), (1, 1, 9, 2, 0, 0), (1, 1, 8, 0, 0, 0), (1, 1, 8, 2, 3, 0), (1 << 31, 1, 8, 2, 0, 0)):
        assert ws(*bad) == -1, bad
    f, b = lib.dgg_group_norm_act_forward, lib.dgg_group_norm_act_backward
    one = 4096   # a pointer that is never read: the checks come first
    fwd = [one, 8, 8, 4, 1, 8, 2, None, None, 1e-5, 1, 0.2, 0, one, None, None, 0, None]
    for k, v in ((0, None), (13, None), (1, -1), (9, -1.0), (9, float("nan")), (10, 3), (12, 7), (6, 3)):
        assert f(*[v if i == k else a for i, a in enumerate(fwd)]) == -1, (k, v)
    for k in (0, 13):                                                          # not an element's address
        assert f(*[one + 2 if i == k else a for i, a in enumerate(fwd)]) == -1, k
    points = [one, 800, 8, 4, 100000, 8, 2, None, None, 1e-5, 1, 0.2, 0, one, None, None, 0, None]
    assert f(*points) == -3 and b"workspace" in lib.dgg_last_error()           # this size needs one
    bwd = [one, 8, 8, one, 8, 8, 4, 1, 8, 2, None, None, 1, 0.2, 0, one, one, None, None, None, 0, None]
    for k, v in ((0, None), (3, None), (15, None), (16, None), (17, one), (18, one), (2, -8)):
        assert b(*[v if i == k else a for i, a in enumerate(bwd)]) == -1, (k, v)


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    y, st = ops.group_norm_act_forward(x, 2, w, w)
    for call in (lambda: ops.group_norm_act_forward(x, 3, w, w), lambda: ops.group_norm_act_forward(x, 2, w[:4], w),
                 lambda: ops.group_norm_act_forward(x, 2, w.half(), w), lambda: ops.group_norm_act_forward(x, 2, w.cpu(), w),
                 lambda: ops.group_norm_act_forward(x.double(), 2, w, w), lambda: ops.group_norm_act_forward(x, 2, w, w, act="relu"),
                 lambda: ops.group_norm_act_forward(x[0], 2, w, w), lambda: ops.group_norm_act_forward(x, 2, w, w, eps=-1.0),
                 lambda: ops.group_norm_act_backward(x[:2], x, 2, w, w, 1e-5, "silu", 0.2, st),
                 lambda: ops.group_norm_act_backward(x.half(), x, 2, w, w, 1e-5, "silu", 0.2, st),
                 lambda: ops.group_norm_act_backward(x, x, 2, w, w, 1e-5, "silu", 0.2, st.float()),
                 lambda: ops.group_norm_act_backward(x, x, 4, w, w, 1e-5, "silu", 0.2, st)):
        with pytest.raises(_lib.DggError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1100, 3, 20, 5), (33000, 2, 6, 2), (1030, 8200, 1, 1), (1, 16384, 64, 1), (3, 128, 4, 4), (3, 129, 4, 4),
                                   (40, 16, 1024, 2)], ids=lambda s: "x".join(map(str, s)))
def test_many_samples_and_long_ones(shape, dtype):
    """More samples than one sum of the parameters' gradients takes; samples whose partial sums a wide workgroup merges."""
    *xs, groups = shape
    check(*data(tuple(xs), dtype, 5)[:2], groups, *data(tuple(xs), dtype, 5)[2:])


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Samples or points 2^31 elements apart, and tensors of more than 2^32 elements, against the same data close together."""
    far = torch.empty((1 << 32) + (1 << 16), dtype=torch.bfloat16, device="cuda")
    for n, s, strides in ((3, 40, (1 << 31, 64, 1)), (1, 3, (64, 1 << 31, 1)), (3, 1, (1 << 31, 64, 1))):
        x, dy, w, b = (t.cuda() for t in data((n, s, 64), torch.bfloat16, 8))
        xf = far.as_strided((n, s, 64), strides)
        xf.copy_(x)
        y, st = ops.group_norm_act_forward(x, 8, w, b)
        yf, sf = ops.group_norm_act_forward(xf, 8, w, b)
        assert torch.equal(y, yf) and torch.equal(st, sf)
        for a, c in zip(ops.group_norm_act_backward(dy, x, 8, w, b, 1e-5, "leaky_relu", 0.2, st),
                        ops.group_norm_act_backward(dy, xf, 8, w, b, 1e-5, "leaky_relu", 0.2, st)):
            assert torch.equal(a, c)
    for s in (1, 4):
        n = ((1 << 32) // 1024 + 64) // s
        x = far[:n * s * 1024].view(n, s, 1024)
        ends = torch.cat([x[:3], x[-3:]])
        ends.copy_(data((6, s, 1024), torch.bfloat16, 9)[0])
        x[:3].copy_(ends[:3])
        x[-3:].copy_(ends[3:])
        y, st = ops.group_norm_act_forward(x, 16)
        small, st_small = ops.group_norm_act_forward(ends, 16)
        assert torch.equal(y[:3], small[:3]) and torch.equal(y[-3:], small[3:]) and torch.equal(st[-3:], st_small[3:])
        dx, _, _ = ops.group_norm_act_backward(x, x, 16, None, None, 1e-5, "leaky_relu", 0.2, st, param_grads=False)
        dx_small, _, _ = ops.group_norm_act_backward(ends, ends, 16, None, None, 1e-5, "leaky_relu", 0.2, st_small, param_grads=False)
        assert torch.equal(dx[:3], dx_small[:3]) and torch.equal(dx[-3:], dx_small[3:])
        del y, dx
    del far
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(6, 1, 35, 7), (50, 1, 99, 11), (9, 1, 39, 3), (4, 1, 31, 1), (70, 1, 515, 5), (3, 1, 2049, 1), (9, 7, 35, 7),
                                   (3, 40, 26, 2), (2, 200, 24, 3), (2, 3000, 64, 4), (2, 9000, 12, 1), (2, 400, 516, 3)],
                         ids=lambda s: "x".join(map(str, s)))
def test_groups_and_addresses_that_no_vector_divides(shape, dtype):
    """Groups whose last vector overlaps the one before it; rows of odd pitch that begin one element into a 16-byte line, and what lies
    beside them."""
    n, s, c, groups = shape
    x, dy, w, b = data((n, s, c), dtype, 12)
    check(x, dy, groups, w, b, act="silu")
    pitch = c + 3 + c % 2
    wide = [torch.full((n, s, pitch), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    xv, dyv = (t[:, :, 1:1 + c] for t in wide)
    xv.copy_(x)
    dyv.copy_(dy)
    check(xv, dyv, groups, w, b)
    flat = torch.full((n * s * c + 5,), 7.0, dtype=dtype, device="cuda")
    odd = flat[1:1 + n * s * c].view(n, s, c)
    odd.copy_(x)
    y, st = ops.group_norm_act_forward(odd, groups, w.cuda(), b.cuda())
    assert torch.equal(y, ops.group_norm_act_forward(x.cuda(), groups, w.cuda(), b.cuda())[0])
    assert all(bool((t[:, :, 0] == 7).all() and (t[:, :, 1 + c:] == 7).all()) for t in wide) and bool((flat[-4:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1100, 5, 64, 4), (600, 32, 64, 32), (700, 9, 24, 3), (5000, 2, 2, 1), (513, 64, 4, 4), (520, 3, 21, 1), (1030, 33, 8, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_many_small_samples(shape, dtype):
    """A few points each: a group in a part of a wave in both directions, samples side by side."""
    n, s, c, groups = shape
    x, dy, w, b = data((n, s, c), dtype, 21)
    _, dx, _, _ = check(x, dy, groups, w, b, act="silu")
    wide = [torch.full((n, s, c + 5), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    xv, dyv = (t[:, :, 3:3 + c] for t in wide)
    xv.copy_(x)
    dyv.copy_(dy)
    check(xv, dyv, groups, None, b)
    st = ops.group_norm_act_forward(xv, groups, w.cuda(), b.cuda(), act="silu")[1]
    only = ops.group_norm_act_backward(dyv, xv, groups, w.cuda(), b.cuda(), 1e-5, "silu", 0.2, st, param_grads=False)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5, 1, 1025, 1), (300, 1, 2048, 2), (70, 1, 4101, 1), (3, 1, 8192, 1), (3, 1, 8193, 1), (1030, 1, 2050, 2), (2, 1, 12001, 1)],
                         ids=lambda s: "x".join(map(str, s)))
def test_long_rows(shape, dtype):
    """A group in a workgroup's registers, on both sides of what fits."""
    n, s, c, groups = shape
    x, dy, w, b = data((n, s, c), dtype, 31)
    check(x, dy, groups, w, b, act="silu")
    wide = torch.full((n, s, c + 3), 7.0, dtype=dtype, device="cuda")
    xv = wide[:, :, 1:1 + c]
    xv.copy_(x)
    check(xv, dy, groups, w, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("c", [1, 7, 64, 515])
def test_groups_of_one_element_have_no_gradient(c, dtype):
    """One point and one channel a group: xh is 0 whatever x is, so dx is exactly 0 — the difference of w dz and its own mean."""
    for n, act in ((1, "none"), (33, "leaky_relu"), (3000, "silu")):
        x, dy, w, b = (t.cuda() for t in data((n, 1, c), dtype, 40 + n))
        y, st = ops.group_norm_act_forward(x, c, w, b, 1e-5, act)
        for ww, bb in ((w, b), (None, None)):
            dx, dw, _ = ops.group_norm_act_backward(dy, x, c, ww, bb, 1e-5, act, 0.2, st)
            assert not dx.any(), (n, act, float(dx.abs().max()))
            assert not dw.any()


# (N, S, C, groups): groups of two to eight elements, rows and points, few samples and many, a last workgroup with fewer groups
SMALL_GROUPS = [(40, 1, 6, 3), (3000, 1, 12, 4), (7, 1, 64, 16), (9, 1, 35, 5), (5, 1, 8, 1), (3, 2, 8, 8), (600, 2, 4, 4), (2, 2, 6, 2), (2000, 3, 2, 1),
                (5, 2, 33, 11), (1, 1, 2, 1), (2, 8, 16, 16), (1, 4, 16, 8), (700, 4, 512, 256), (1100, 8, 96, 96), (2, 2, 2052, 513), (3, 7, 515, 515),
                (1, 2, 8192, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SMALL_GROUPS, ids=lambda s: "x".join(map(str, s)))
def test_dx_of_small_groups_is_rounded_once(shape, dtype):
    """In a group of a few elements the three terms of dx cancel nearly (two elements: to eps / (var + eps) of them), so they have to be
    added up in 64 bits.  Without an activation dz is dy, every sum and product is a 64-bit one (2^-40 of the terms is far above what the
    roundings of 2^-53 make of 8 of them with x within a few deviations of 0), and what is left is the rounding to fp32 and that to
    the output type."""
    n, s, c, g = shape
    x, dy, w, b = data((n, s, c), dtype, 50 + n)
    for ww in (w, None):
        xd, dyd, wd = x.cuda(), dy.cuda(), None if ww is None else ww.cuda()
        y, st = ops.group_norm_act_forward(xd, g, wd, None, 1e-5, "none")
        dx, _, _ = ops.group_norm_act_backward(dyd, xd, g, wd, None, 1e-5, "none", 0.2, st)
        r = reference(x, dy, g, ww, None, 1e-5, "none", 0.2)
        xh = (r["z"] / (torch.ones(c) if ww is None else ww).double().view(g, -1)).abs()
        wdz = (dy.double().reshape(r["dx"].shape) * (torch.ones(c) if ww is None else ww).double().view(g, -1)).abs()
        terms = r["rstd"] * (wdz + wdz.mean((1, 3), keepdim=True) + xh * (wdz * xh).mean((1, 3), keepdim=True))
        close(dx, r["dx"], half_step(dtype, r["dx"]) + U * r["dx"].abs() + 2.0 ** -40 * terms, "dx")


def test_launches_beyond_2_32_threads_are_refused_without_a_gpu():
    lib = _lib.lib()
    ws = lib.dgg_group_norm_workspace_bytes
    for shape in ((1 << 24, 9000, 1, 1), (1 << 20, 9000, 16, 16), (1, 9000, (1 << 24) - 1, 1)):
        for backward in (0, 1):
            assert ws(*shape, _lib.BF16, backward) == -1 and b"2^32" in lib.dgg_last_error(), shape
        n, s, c, g = shape
        one = 4096   # never read: the checks come first
        assert lib.dgg_group_norm_act_forward(one, s * c, c, n, s, c, g, None, None, 1e-5, 1, 0.2, _lib.BF16, one, None, one, 1 << 62, None) == -1
    assert ws((1 << 22) - 1, 9000, 1, 1, _lib.BF16, 1) > 0 and ws((1 << 26) + 5, 33, 1, 1, _lib.BF16, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n,s,first", [((1 << 26) + 5, 33, ((1 << 32) - 1024) // 64), ((1 << 24) + 3, 300, ((1 << 32) - 1024) // 320)],
                         ids=["part of a wave", "workgroup"])
def test_more_samples_than_a_launch_has_threads(n, s, first):
    """2^32 threads and more go in several launches: samples at both ends and where a second launch begins (`first`, in the forward pass)."""
    x = torch.empty((n, s, 1), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    dy = torch.zeros_like(x)
    at = torch.tensor([0, 1, 2, first - 2, first - 1, first, first + 1, n // 2, n - 2, n - 1], device="cuda")
    small, dsmall, w, b = data((len(at), s, 1), torch.bfloat16, 60)
    x[at], dy[at] = small.cuda(), dsmall.cuda()
    y, st = ops.group_norm_act_forward(x, 1, w.cuda(), b.cuda())
    r = reference(small, dsmall, 1, w, b, 1e-5, "leaky_relu", 0.2)
    close(y[at], r["y"], half_step(x.dtype, r["y"]) + (8 + r["z"].abs()) * U * r["y"].abs(), "y")
    close(st[at][..., 1], r["rstd"].reshape(-1, 1), 1e-12 * r["rstd"].reshape(-1, 1), "rstd")
    assert bool((st[..., 1] > 0.25).all()) and not bool((st[..., 1] > 1e3).any())       # every sample has its own
    del y
    dx, dw, db = ops.group_norm_act_backward(dy, x, 1, w.cuda(), b.cuda(), 1e-5, "leaky_relu", 0.2, st)
    close(dx[at], r["dx"], half_step(x.dtype, r["dx"]) + r["dx_tol"], "dx")
    close(dw, r["dw"], r["dw_tol"] + U * r["dw"].abs(), "dweight")                        # dy is zero in every other sample
    close(db, r["db"], r["db_tol"] + U * r["db"].abs(), "dbias")
    del x, dy, dx, st
    torch.cuda.empty_cache()
