"""Newton-Schulz orthogonalisation (ops.orthogonalize) and the Muon step (ops.muon_step) against the iteration in 64 bits on the CPU,
at the sizes, layouts and values where they can go wrong, and their refusals.

Tolerances.  A step multiplies operands of 22 bits (two fp16 planes: 2^-23 of a value at most, the dropped lo lo 2^-22 of a term) and
sums in fp32, and b A + c A^2 is a difference of terms a few times its size: 2^-21 of |X| is allowed a step.  Later steps pass an error on
with the iteration's derivative, whose largest value from X_0 on is kappa = max(|p'(s)|, |p(s) / s|) over the singular values s of X_0
(p: the composed polynomial; 0 belongs to them where the rank is short).  So |error|_F <= 2^-21 (steps |X|_F + kappa |X_0|_F); a single
element is allowed 20 times the root mean square of that.  Outputs of 16 bits: half a step of the type more."""
import math

import pytest
import torch

from dex_gan_grasp_amd import _lib, ops

COEF = ops.NS_COEFFICIENTS
EPS = 1e-7
U = 2.0 ** -24


def reference(g, steps=5, coef=COEF, eps=EPS):
    """The iteration in doubles on the CPU for one matrix, and the Frobenius error allowed."""
    g = g.double().cpu()
    turned = g.shape[0] > g.shape[1]
    x = g.t() if turned else g
    x = x / (x.norm() + eps)
    rows = [coef] * steps if not hasattr(coef[0], "__len__") else coef
    s = torch.linalg.svdvals(x)
    if x.shape[0] > 1:
        s = torch.cat([s, torch.zeros(1, dtype=torch.float64)])
    p, dp, over, x0 = s.clone(), torch.ones_like(s), torch.ones_like(s), float(x.norm())
    for a, b, c in rows:
        dp = dp * (a + 3 * b * p ** 2 + 5 * c * p ** 4)
        over = over * (a + b * p ** 2 + c * p ** 4)      # p(s) / s, also at 0
        p = p * (a + b * p ** 2 + c * p ** 4)
        gram = x @ x.t()
        x = a * x + (b * gram + c * gram @ gram) @ x
    kappa = float(torch.maximum(dp.abs(), over.abs()).max())
    tol = 2.0 ** -21 * (steps * float(x.norm()) + kappa * x0)
    return (x.t() if turned else x), tol


def close(got, g, dtype=torch.float32, **kw):
    ref, tol = reference(g, **kw)
    got = got.double().cpu()
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else U
    err = (got - ref).abs()
    rms = tol / math.sqrt(ref.numel())
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    assert float((got - ref).norm()) <= tol + half * float(ref.norm()) + tiny * math.sqrt(ref.numel()), (
        float((got - ref).norm()), tol, float(ref.norm()))
    assert bool((err <= 20 * rms + half * ref.abs() + tiny).all()), float((err / (20 * rms + half * ref.abs() + tiny)).max())


def matrix(rows, cols, seed, dtype=torch.float32, kind="gradient"):
    g = torch.Generator().manual_seed(seed)
    if kind == "gradient":      # dy^T x over a batch of 300, scales spread over a decade
        dy = torch.randn(300, rows, generator=g) * torch.logspace(0, -1, rows)
        m = dy.t() @ torch.randn(300, cols, generator=g) / 300
    elif kind == "low rank":
        m = torch.randn(rows, 3, generator=g) @ torch.randn(3, cols, generator=g)
    else:
        m = torch.randn(rows, cols, generator=g)
    return m.to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (1, 300), (2, 2), (12, 512), (3, 512), (31, 33), (63, 65), (64, 64), (65, 63), (66, 200), (128, 128),
          (129, 257), (200, 100), (257, 771), (512, 256), (320, 700), (100, 4101), (4613, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_matches_the_iteration(shape):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        g = matrix(*shape, seed=sum(shape), dtype=dtype)
        out = ops.orthogonalize(g.cuda())
        assert out.dtype == dtype and out.shape == g.shape and out.is_contiguous()
        close(out, g, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["low rank", "normal"])
@pytest.mark.parametrize("shape", [(40, 90), (256, 512), (300, 130)], ids=lambda s: "%dx%d" % s)
def test_spectra(shape, kind):
    g = matrix(*shape, seed=3, kind=kind)
    close(ops.orthogonalize(g.cuda()), g)
    if kind == "normal":        # what it is for: singular values near 1
        s = torch.linalg.svdvals(ops.orthogonalize(g.cuda()).double().cpu())
        assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.gpu
def test_scales_and_special_values():
    g = matrix(70, 130, 4)
    for scale in (1e-4, 1e-12, 1e-16, 1e15, 1e30):      # (from 1e-12 down eps is larger than the norm)
        close(ops.orthogonalize((g * scale).cuda()), g * scale)
    assert not ops.orthogonalize(torch.zeros(70, 130, device="cuda")).any()
    spike = torch.zeros(70, 130)
    spike[5, 7] = -3.0
    close(ops.orthogonalize(spike.cuda()), spike)
    close(ops.orthogonalize((g * 1e-30).cuda(), eps=0.0), g * 1e-30, eps=0.0)
    stack = torch.stack([g, g, g, g])
    stack[1, 69, 129] = float("nan")
    stack[2, 0, 3] = float("inf")
    out = ops.orthogonalize(stack.cuda())
    one = ops.orthogonalize(g.cuda())
    assert torch.equal(out[0], one) and torch.equal(out[3], one) and out[1].isnan().all() and out[2].isnan().all()


@pytest.mark.gpu
def test_steps_and_coefficients():
    g = matrix(48, 100, 6)
    for steps in (1, 2, 10):
        close(ops.orthogonalize(g.cuda(), steps), g, steps=steps)
    rows = [(3.0, -3.2, 1.2), (2.5, -2.0, 0.6), (1.875, -1.25, 0.375)]
    close(ops.orthogonalize(g.cuda(), 3, rows), g, steps=3, coef=rows)
    close(ops.orthogonalize(g.cuda(), 8, (1.5, -0.5, 0.0)), g, steps=8, coef=(1.5, -0.5, 0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(31, 200), (64, 100), (128, 128), (300, 170)], ids=lambda s: "%dx%d" % s)
def test_operands_keep_22_bits(shape):
    """With X <- X in every step what is left of each is taking X apart into two planes and putting it together again: hi is off by
    2^-12 of a value at most, lo by 2^-12 of that, so 2^-23 a step (one more for the common factor) — element by element, where a hi
    and a lo of two different roundings would differ by 2^-11."""
    g = matrix(*shape, seed=11)
    out = ops.orthogonalize(g.cuda(), 10, (1.0, 0.0, 0.0)).double().cpu()
    ref = g.double() / (g.double().norm() + EPS)
    assert bool(((out - ref).abs() <= 11 * 2.0 ** -23 * ref.abs() + 2.0 ** -38).all())   # 2^-38: fp16's smallest step under 2^14


@pytest.mark.gpu
def test_stacks_lists_and_strides():
    stack = torch.stack([matrix(33, 65, s) for s in range(5)])
    out = ops.orthogonalize(stack.cuda())
    for o, g in zip(out, stack):
        close(o, g)
    # more entries than one set of launches takes, of all shapes; an empty one among them
    shapes = [(1 + 7 * i % 40, 1 + 13 * i % 90) for i in range(19)] + [(0, 5), (300, 200)]
    many = [matrix(*s, seed=i) for i, s in enumerate(shapes)]
    outs = ops.orthogonalize([m.cuda() for m in many])
    for o, g in zip(outs, many):
        assert o.shape == g.shape
        if g.numel():
            close(o, g)
    g = matrix(40, 100, 8)
    want = ops.orthogonalize(g.cuda())
    wide = torch.full((40, 131), 9.0, device="cuda")
    wide[:, 17:117] = g.cuda()
    assert torch.equal(ops.orthogonalize(wide[:, 17:117]), want)
    assert torch.equal(ops.orthogonalize(g.t().contiguous().cuda().t()), want)
    assert torch.equal(ops.orthogonalize(stack.cuda().transpose(0, 1).contiguous().transpose(0, 1)), out)
    row = matrix(1, 100, 9)
    close(ops.orthogonalize(row.cuda().expand(6, 100)), row.expand(6, 100))


def muon_reference(w, g, m, lr, mu, nesterov, wd, f, gs):
    m64 = mu * m.double() + gs * g.double()
    ref, tol = reference(gs * g.double() + mu * m64 if nesterov else m64)
    return (1 - lr * wd) * w.double() - lr * f * ref, m64, lr * f * tol


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,adjust,gs", [(True, "spectral", 1.0), (False, "match_rms", 0.125)], ids=["nesterov", "plain"])
def test_muon_step(nesterov, adjust, gs):
    shapes = [(256, 300), (512, 256), (12, 512), (1, 9), (65, 64), (130, 40)]
    lr, mu, wd = 0.02, 0.95, 0.1
    ws = [matrix(*s, seed=1, kind="normal") for s in shapes]
    gs_ = [matrix(*s, seed=2) for s in shapes]
    ms = [matrix(*s, seed=3) for s in shapes]
    # parameters as column blocks of wider tensors: what lies beside them stays
    wide = [torch.full((s[0], s[1] + 5), 4.0, device="cuda") for s in shapes]
    dw = [t[:, 2:2 + s[1]].copy_(w) for t, s, w in zip(wide, shapes, ws)]
    dg, dm = [t.cuda() for t in gs_], [t.cuda() for t in ms]
    ops.muon_step(dw, dg, dm, lr, mu, nesterov, wd, adjust=adjust, grad_scale=gs)
    for s, w, g, m, nw, ng, nm, t in zip(shapes, ws, gs_, ms, dw, dg, dm, wide):
        f = math.sqrt(max(1.0, s[0] / s[1])) if adjust == "spectral" else 0.2 * math.sqrt(max(s))
        rw, rm, tol = muon_reference(w, g, m, lr, mu, nesterov, wd, f, gs)
        assert torch.equal(ng.cpu(), g)
        # M: mu rounded to fp32, one product and one sum rounded
        assert bool(((nm.cpu().double() - rm).abs() <= 3 * U * (m.double().abs() + gs * g.double().abs() + rm.abs())).all())
        err = (nw.cpu().double() - rw).abs()
        # W: decay and step rounded, one fma; u's own roundings (3 U) pass through the iteration like its 2^-21 of a step
        assert float(err.norm()) <= 2 * tol + 4 * U * float(w.norm()) and bool((err <= 40 * tol / math.sqrt(w.numel())
                                                                                 + 4 * U * (w.double().abs() + rw.abs())).all())
        assert bool((t[:, :2] == 4).all()) and bool((t[:, 2 + s[1]:] == 4).all())


@pytest.mark.gpu
def test_muon_of_a_zero_gradient_and_of_stacks():
    w = torch.randn(3, 20, 30, device="cuda")
    m = torch.zeros_like(w)
    was = w.clone()
    ops.muon_step([w], [torch.zeros_like(w)], [m], 0.1, weight_decay=0.5)
    assert not m.any() and bool(((w - 0.95 * was).abs() <= 2 * U * was.abs()).all())
    g = torch.stack([matrix(20, 30, s) for s in range(3)]).cuda()
    one = [t.clone() for t in w]
    ops.muon_step([w], [g], [m], 0.1)
    for i in range(3):
        ops.muon_step([one[i]], [g[i]], [torch.zeros(20, 30, device="cuda")], 0.1)
        assert torch.equal(one[i], w[i])


@pytest.mark.gpu
def test_other_streams_and_graph_replays():
    shapes = [(200, 300), (12, 512), (256, 64)]
    gs = [matrix(*s, seed=5).cuda() for s in shapes]
    want = ops.orthogonalize(gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.orthogonalize(gs)
        again = ops.orthogonalize(gs)
    both = ops.orthogonalize(gs)          # beside the other stream's: a workspace of its own
    torch.cuda.synchronize()
    for e, a, b, c in zip(want, got, again, both):
        assert torch.equal(e, a) and torch.equal(e, b) and torch.equal(e, c)
    ws, ms = [torch.randn_like(g) for g in gs], [torch.zeros_like(g) for g in gs]
    ew, em = [w.clone() for w in ws], [m.clone() for m in ms]
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step(ws, gs, ms, 0.02, weight_decay=0.01)
    with torch.cuda.graph(second):
        out = ops.orthogonalize(gs)
    for k in range(4):
        for g, s in zip(gs, shapes):
            g.copy_(matrix(*s, seed=30 + k))
        graph.replay()
        second.replay()
        ops.muon_step(ew, gs, em, 0.02, weight_decay=0.01)
        eager = ops.orthogonalize(gs)
        torch.cuda.synchronize()
        for a, b in zip(ws + ms + list(out), ew + em + list(eager)):
            assert torch.equal(a, b), k


def test_refusals_without_a_gpu():
    with pytest.raises(_lib.DggError):
        ops.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(_lib.DggError):
        ops.muon_step([torch.zeros(4, 4)], [torch.zeros(4, 4)], [torch.zeros(4, 4)], 0.1)
    lib = _lib.lib()
    C = _lib.C
    coef = (C.c_double * 15)(*(COEF * 5))

    def mat(**kw):
        m = (_lib.Matrix * 1)()
        base = dict(in_=4096, out=4096, momentum=4096, batch=1, rows=8, cols=8, ld_in=8, ld_out=8, ld_momentum=8)
        for k, v in {**base, **kw}.items():
            setattr(m[0], k, v)
        return m

    need = lib.dgg_orthogonalize_workspace_bytes(mat(), 1)
    assert need > 0 and lib.dgg_orthogonalize_workspace_bytes(mat(), 0) == -1
    for bad in (dict(rows=0), dict(cols=-1), dict(batch=0), dict(rows=16385, cols=16385), dict(cols=(1 << 20) + 1), dict(batch=1 << 30)):
        assert lib.dgg_orthogonalize_workspace_bytes(mat(**bad), 1) == -1, bad

    def orth(m=None, dtype=0, c=coef, steps=5, eps=1e-7, ws=4096, n=need):
        return lib.dgg_orthogonalize(mat() if m is None else m, 1, dtype, c, steps, eps, ws, n, None)

    def muon(m=None, lr=0.1, mu=0.9, adjust=0, gs=1.0):
        return lib.dgg_muon_step(mat() if m is None else m, 1, lr, mu, 1, 0.0, adjust, gs, coef, 5, 1e-7, 4096, 0, None)

    assert orth(dtype=3) == orth(c=None) == orth(steps=0) == orth(steps=17) == orth(eps=-1.0) == orth(eps=float("nan")) == -1
    assert orth(c=(C.c_double * 15)(*([9.0] * 15))) == -1                       # iterates that run away
    assert orth(c=(C.c_double * 15)(*([float("nan")] * 15))) == -1
    for bad in (dict(in_=None), dict(out=None), dict(ld_in=7), dict(ld_out=7), dict(in_stride=-1)):
        assert orth(mat(**bad)) == -1, bad
    assert orth(ws=None) == orth(ws=4100) == orth(n=need - 1) == -3
    assert muon(adjust=2) == muon(lr=float("inf")) == muon(mu=float("nan")) == muon(gs=float("nan")) == -1
    assert muon(mat(momentum=None)) == muon(mat(ld_momentum=7)) == -1
    assert muon() == -3                                                         # no workspace


@pytest.mark.gpu
def test_refusals():
    g = torch.zeros(4, 6, device="cuda")
    f = torch.zeros(4, 6, device="cuda")
    for call in (lambda: ops.orthogonalize(g[0]), lambda: ops.orthogonalize(g.double()), lambda: ops.orthogonalize([g, g.half()]),
                 lambda: ops.orthogonalize([g, g.cpu()]), lambda: ops.orthogonalize(g, 0), lambda: ops.orthogonalize(g, 17),
                 lambda: ops.orthogonalize(g, 3, [COEF, COEF]), lambda: ops.orthogonalize(g, 5, (30.0, 0.0, 0.0)),
                 lambda: ops.muon_step([g], [f], [], 0.1), lambda: ops.muon_step([g], [f[:2]], [f], 0.1),
                 lambda: ops.muon_step([g], [f.half()], [f], 0.1), lambda: ops.muon_step([g.t()], [f.t()], [f.t()], 0.1),
                 lambda: ops.muon_step([g], [f], [f], 0.1, adjust="none"),
                 lambda: ops.muon_step([g[:1].expand(4, 6)], [f], [f], 0.1), lambda: ops.muon_step([g], [f], [g], 0.1),
                 lambda: ops.muon_step([g, g], [f, f], [torch.zeros_like(g), torch.zeros_like(g)], 0.1)):
        with pytest.raises(_lib.DggError):
            call()
    assert ops.orthogonalize([]) == []


def test_overlaps_are_refused_without_a_gpu():
    """What a call writes may overlap nothing else in it.  (Layouts that share a buffer and are accepted: the test below.)"""
    lib, C = _lib.lib(), _lib.C
    coef = (C.c_double * 15)(*(COEF * 5))
    base = 1 << 20

    def call(*mats, muon=True, dtype=0):
        arr = (_lib.Matrix * len(mats))()
        for m, kw in zip(arr, mats):
            d = dict(in_=base, out=2 * base, momentum=3 * base, batch=1, rows=8, cols=8, ld_in=8, ld_out=8, ld_momentum=8)
            for k, v in {**d, **kw}.items():
                setattr(m, k, v)
        n = lib.dgg_orthogonalize_workspace_bytes(arr, len(mats))
        if muon:
            return lib.dgg_muon_step(arr, len(mats), 0.1, 0.9, 1, 0.0, 0, 1.0, coef, 5, 1e-7, 4096, n, None)
        return lib.dgg_orthogonalize(arr, len(mats), dtype, coef, 5, 1e-7, 4096, n, None)

    other = dict(in_=4 * base, out=5 * base, momentum=6 * base)
    for bad in ([dict(in_=3 * base)], [dict(in_=2 * base)], [dict(momentum=2 * base)], [dict(momentum=2 * base + 252)],
                [dict(in_=3 * base - 252)], [{}, {}], [{}, dict(other, out=2 * base + 4)], [{}, dict(other, in_=3 * base)],
                [dict(batch=2, in_stride=64, out_stride=63, momentum_stride=64)], [dict(batch=2, in_stride=64, out_stride=64)],
                [dict(batch=2, in_stride=64, out_stride=64, momentum_stride=8)],
                [dict(ld_out=16), dict(other, out=2 * base + 28, ld_out=16)], [dict(ld_out=16), dict(other, out=2 * base + 32, ld_out=24)],
                [dict(ld_out=16), dict(other, out=2 * base + 40, ld_out=16)]):
        assert call(*bad) == -1, bad
        assert b"overlaps" in lib.dgg_last_error(), bad
    for bad in ([dict(out=base + 4)], [dict(out=base, ld_out=9)], [{}, {}], [{}, dict(in_=2 * base, out=5 * base)]):
        assert call(*bad, muon=False) == -1, bad
        assert b"overlaps" in lib.dgg_last_error(), bad


@pytest.mark.gpu
def test_layouts_that_share_a_buffer():
    """Parameters that are column blocks of one buffer, stacks whose matrices lie side by side, one gradient for several matrices."""
    g = torch.stack([matrix(20, 30, s) for s in range(3)]).cuda()
    want = [torch.ones(20, 30, device="cuda") for _ in range(3)]
    mom = [torch.zeros(20, 30, device="cuda") for _ in range(3)]
    for i in range(3):
        ops.muon_step([want[i]], [g[i]], [mom[i]], 0.1)
    wide = torch.ones(20, 100, device="cuda")
    ops.muon_step([wide[:, 30 * i:30 * i + 30] for i in range(3)], list(g), [torch.zeros(20, 30, device="cuda") for _ in range(3)], 0.1)
    beside, m = torch.ones(20, 3, 30, device="cuda"), torch.zeros(20, 3, 30, device="cuda")
    ops.muon_step([beside.transpose(0, 1)], [g], [m.transpose(0, 1)], 0.1)
    for i in range(3):
        assert torch.equal(wide[:, 30 * i:30 * i + 30], want[i]) and torch.equal(beside[:, i], want[i]) and torch.equal(m[:, i], mom[i])
    assert bool((wide[:, 90:] == 1).all())
    two = torch.ones(2, 20, 30, device="cuda")
    ops.muon_step([two], [g[:1].expand(2, 20, 30)], [torch.zeros_like(two)], 0.1)
    assert torch.equal(two[0], want[0]) and torch.equal(two[1], want[0])
    w, m = torch.ones(20, 30, device="cuda"), torch.zeros(20, 30, device="cuda")
    for call in (lambda: ops.muon_step([w], [m], [m], 0.1), lambda: ops.muon_step([w], [w], [m], 0.1),
                 lambda: ops.muon_step([w, w[:10]], [g[0], g[0][:10]], [m, torch.zeros(10, 30, device="cuda")], 0.1)):
        with pytest.raises(_lib.DggError):
            call()
    assert bool((w == 1).all()) and not m.any()


# short sides up to 64 beside long ones: on both sides of what one workgroup holds (512 and 192 columns, 256 and 128 of a longer one) and
# of the longest
NARROW = [(1, 513), (12, 700), (32, 512), (32, 513), (32, 769), (33, 193), (64, 1024), (64, 1025), (5000, 7), (4108, 64), (32, 16384),
          (32, 16385), (64, 6144), (64, 6145)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", NARROW, ids=lambda s: "%dx%d" % s)
def test_narrow_matrices(shape):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        g = matrix(*shape, seed=sum(shape), dtype=dtype)
        close(ops.orthogonalize(g.cuda()), g, dtype)
    g = matrix(*shape, seed=7)
    out = ops.orthogonalize(g.cuda(), 10, (1.0, 0.0, 0.0)).double().cpu()      # (test_operands_keep_22_bits)
    ref = g.double() / (g.double().norm() + EPS)
    assert bool(((out - ref).abs() <= 11 * 2.0 ** -23 * ref.abs() + 2.0 ** -38).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(20, 900), (1500, 50)], ids=lambda s: "%dx%d" % s)
def test_narrow_scales_and_special_values(shape):
    g = matrix(*shape, seed=4)
    for scale in (1e-4, 1e-12, 1e-16, 1e15, 1e30):
        close(ops.orthogonalize((g * scale).cuda()), g * scale)
    assert not ops.orthogonalize(torch.zeros(*shape, device="cuda")).any()
    spike = torch.zeros(*shape)
    spike[5, 7] = -3.0                                       # every other workgroup's columns are zero
    close(ops.orthogonalize(spike.cuda()), spike)
    uneven = g.clone()                                       # columns whose powers of two lie far apart
    (uneven if shape[1] > shape[0] else uneven.t())[:, :300] *= 1e-18
    close(ops.orthogonalize(uneven.cuda()), uneven)
    close(ops.orthogonalize((g * 1e-30).cuda(), eps=0.0), g * 1e-30, eps=0.0)
    stack = torch.stack([g, g, g, g])
    stack[1, -1, -1] = float("nan")
    stack[2, 0, 3] = float("inf")
    out = ops.orthogonalize(stack.cuda())
    one = ops.orthogonalize(g.cuda())
    assert torch.equal(out[0], one) and torch.equal(out[3], one) and out[1].isnan().all() and out[2].isnan().all()
    pitch = torch.full((shape[0], shape[1] + 9), 4.0, device="cuda")
    pitch[:, 3:3 + shape[1]] = g.cuda()
    assert torch.equal(ops.orthogonalize(pitch[:, 3:3 + shape[1]]), one)
    for steps in (1, 2, 9):
        close(ops.orthogonalize(g.cuda(), steps), g, steps=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(20, 900), (1000, 64), (12, 512), (3, 4)], [(33, 700)] * 18, [(40, 600), (100, 130), (5, 9)],
                                    [(8, 30)] * 17 + [(30, 800)], [(8, 30)] * 17 + [(100, 200)]],
                         ids=["narrow and small", "more than 16", "with general ones", "small apart", "small apart, general"])
def test_muon_step_of_narrow_and_mixed_matrices(shapes):
    lr, mu, wd = 0.02, 0.9, 0.1
    ws = [matrix(*s, seed=i, kind="normal") for i, s in enumerate(shapes)]
    gs = [matrix(*s, seed=50 + i) for i, s in enumerate(shapes)]
    ms = [matrix(*s, seed=90 + i) for i, s in enumerate(shapes)]
    wide = [torch.full((s[0], s[1] + 5), 4.0, device="cuda") for s in shapes]
    dw = [t[:, 2:2 + s[1]].copy_(w) for t, s, w in zip(wide, shapes, ws)]
    dg, dm = [t.cuda() for t in gs], [t.cuda() for t in ms]
    graph, side = torch.cuda.CUDAGraph(), [(w.clone(), m.clone()) for w, m in zip(dw, dm)]
    with torch.cuda.graph(graph):
        ops.muon_step([w for w, _ in side], dg, [m for _, m in side], lr, mu, weight_decay=wd)
    for k in range(3):
        before = [(w.cpu(), m.cpu()) for w, m in zip(dw, dm)]
        ops.muon_step(dw, dg, dm, lr, mu, weight_decay=wd)
        graph.replay()
        torch.cuda.synchronize()
        for (w, m), g, nw, nm, (gw, gm), t in zip(before, gs, dw, dm, side, wide):
            s = w.shape
            rw, rm, tol = muon_reference(w, g, m, lr, mu, True, wd, math.sqrt(max(1.0, s[0] / s[1])), 1.0)
            assert bool(((nm.cpu().double() - rm).abs() <= 3 * U * (m.double().abs() + g.double().abs() + rm.abs())).all())
            err = (nw.cpu().double() - rw).abs()
            assert float(err.norm()) <= 2 * tol + 4 * U * float(w.norm())
            assert bool((err <= 40 * tol / math.sqrt(w.numel()) + 4 * U * (w.double().abs() + rw.abs())).all())
            assert torch.equal(gw, nw) and torch.equal(gm, nm), k
            assert bool((t[:, :2] == 4).all()) and bool((t[:, 2 + s[1]:] == 4).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1600, 1700), (1100, 700), (66, 20000)], ids=lambda s: "%dx%d" % s)
def test_large_matrices(shape):
    g = matrix(*shape, seed=3)
    close(ops.orthogonalize(g.cuda()), g)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Matrices 2^31 elements apart; rows further apart than a pitch may be are copied, or refused where they are written."""
    far = torch.empty((1 << 32) + (1 << 17), dtype=torch.float32, device="cuda")
    for shape in ((20, 30), (40, 700), (70, 200)):
        g = torch.stack([matrix(*shape, seed=s) for s in range(3)]).cuda()
        view = far.as_strided(g.shape, (1 << 31, shape[1], 1))
        view.copy_(g)
        assert torch.equal(ops.orthogonalize(view), ops.orthogonalize(g))
        w, m = torch.ones_like(g), torch.zeros_like(g)
        ops.muon_step([w], [g], [m], 0.1)
        view.fill_(1.0)
        fm = torch.zeros_like(g)
        ops.muon_step([view], [g], [fm], 0.1)
        assert torch.equal(view, w) and torch.equal(fm, m)
    rows = far.as_strided((3, 50), (1 << 31, 1))
    rows.copy_(g[0, :3, :50])
    assert torch.equal(ops.orthogonalize(rows), ops.orthogonalize(g[0, :3, :50].contiguous()))
    with pytest.raises(_lib.DggError):
        ops.muon_step([rows], [g[0, :3, :50]], [torch.zeros(3, 50, device="cuda")], 0.1)
    with pytest.raises(_lib.DggError):
        ops.orthogonalize(far[:(1 << 32) + 5].view(1, -1))
    with pytest.raises(_lib.DggError):
        ops.orthogonalize(g, 1 << 33)
    del far, view, rows
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(32, 500), (60, 2000), (512, 1025), (700, 300)], ids=lambda s: "%dx%d" % s)
def test_a_small_weight_decay_is_the_one_asked_for(shape):
    """lr wd = 5e-8 and half of it — the trainers' defaults — lie below the spacing of fp32 under 1: the parameters move by it on average,
    beside the update that rounds each of them one way or the other.  sum sign(w) (w - w' - update) / sum |w| is lr wd, off by
      the rounding of w' (one, so at most half a step of it; over n parameters six times the root mean square of a step / sqrt 12: the
        update, many steps long and the same function of no parameter, spreads it evenly),
      the update's own error, |error|_F <= lr f tol, so sqrt(n) lr f tol in the sum."""
    w = matrix(*shape, seed=1, kind="normal")
    g = matrix(*shape, seed=2, kind="normal")
    for lr in (1e-4, 0.5e-4):
        wd = 5e-4
        p, m = w.cuda(), torch.zeros(shape, device="cuda")
        ops.muon_step([p], [g.cuda()], [m], lr, 0.0, True, wd, adjust="match_rms")
        ref, tol = reference(g)
        f = 0.2 * math.sqrt(max(shape))
        new = p.cpu().double()
        total = float(w.double().abs().sum())
        decay = float((w.double().sign() * (w.double() - new - lr * f * ref)).sum()) / total
        step = torch.ldexp(torch.ones(shape, dtype=torch.float64), torch.frexp(new)[1] - 24)
        allowed = (6 * float(((step ** 2).sum() / 12).sqrt()) + math.sqrt(w.numel()) * lr * f * tol) / total
        assert allowed < 0.12 * lr * wd, (allowed, lr * wd)
        assert abs(decay - lr * wd) <= allowed, (decay / (lr * wd), allowed / (lr * wd))


@pytest.mark.gpu
def test_infinite_parameters_stay_infinite():
    for shape in ((20, 30), (30, 900), (100, 130)):
        w = torch.ones(shape, device="cuda")
        w[3, 4], w[5, 6] = float("inf"), -float("inf")
        for wd in (0.0, 0.1):
            ops.muon_step([w], [matrix(*shape, seed=3).cuda()], [torch.zeros(shape, device="cuda")], 0.1, weight_decay=wd)
            assert w[3, 4] == float("inf") and w[5, 6] == -float("inf") and int(w.isfinite().sum()) == w.numel() - 2


def test_stacks_beyond_2_32_threads_are_refused_without_a_gpu():
    lib = _lib.lib()
    for kw in (dict(batch=1 << 18, rows=1, cols=16384), dict(batch=1 << 12, rows=1 << 20, cols=1), dict(batch=1 << 11, rows=2, cols=1 << 20)):
        mats = (_lib.Matrix * 2)()
        for m, d in zip(mats, (dict(batch=1, rows=8, cols=8), kw)):
            for k, v in dict(in_=4096, out=4096, momentum=4096, ld_in=1 << 20, ld_out=1 << 20, ld_momentum=1 << 20, **d).items():
                setattr(m, k, v)
        assert lib.dgg_orthogonalize_workspace_bytes(mats, 2) == -1 and b"2^32" in lib.dgg_last_error(), kw
    mats[1].batch = (1 << 20) // 2      # half of the threads' limit
    mats[1].rows = mats[1].cols = 65
    assert lib.dgg_orthogonalize_workspace_bytes(mats, 2) > 0


@pytest.mark.gpu
def test_stacks_that_need_more_than_one_launch():
    """Five stacks of 2^20 matrices of one element: 1024 threads a matrix are 5 x 2^30."""
    gen = torch.Generator("cuda").manual_seed(1)
    gs = [torch.empty(1 << 20, 1, 1, device="cuda").uniform_(0.5, 2.0, generator=gen) for _ in range(5)]
    gs[4].neg_()
    ref, tol = reference(torch.ones(1, 1))              # (eps, 2e-7 of the smallest, makes less of a difference than the other roundings)
    ref, tol = ref.item(), 20 * tol
    for g, o in zip(gs, ops.orthogonalize(gs)):
        assert bool(((o * g.sign() - ref).abs() <= tol).all())
    ws, ms = [torch.ones_like(g) for g in gs], [torch.zeros_like(g) for g in gs]
    ops.muon_step(ws, gs, ms, 0.5, 0.0)
    for w, m, g in zip(ws, ms, gs):
        assert bool(((w - (1 - 0.5 * ref * g.sign())).abs() <= tol).all()) and torch.equal(m, g)


@pytest.mark.gpu
def test_autograd_knows_what_a_muon_step_wrote():
    w = torch.randn(20, 30, device="cuda", requires_grad=True)
    m = torch.zeros(20, 30, device="cuda")
    loss = (w * w).sum()
    g, = torch.autograd.grad(loss, w, retain_graph=True)
    versions = w._version, m._version, g._version
    ops.muon_step([w], [g], [m], 0.1)
    assert w._version > versions[0] and m._version > versions[1] and g._version == versions[2]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w)
    (w * w).sum().backward()
    assert torch.equal(w.grad, 2 * w.detach())
    flat = torch.zeros(2, 20, 30, device="cuda")        # a view's base, and what has no versions
    ops.muon_step([flat[0]], [g], [m], 0.1)
    assert flat._version > 0
    with torch.inference_mode():
        w = torch.ones(20, 30, device="cuda")
        ops.muon_step([w], [g], [torch.zeros_like(w)], 0.1)
    assert bool((w != 1).any())


@pytest.mark.gpu
def test_stacks_that_alternate_and_single_rows_are_apart():
    """Stacks whose matrices alternate in one buffer, a matrix between those of a stack, rows of a buffer beside a column block of it."""
    g = torch.stack([matrix(20, 30, s) for s in range(4)]).cuda()
    want = [torch.ones(20, 30, device="cuda") for _ in range(4)]
    for i in range(4):
        ops.muon_step([want[i]], [g[i]], [torch.zeros(20, 30, device="cuda")], 0.1)
    both, mom = torch.ones(2, 2, 20, 30, device="cuda"), torch.zeros(2, 2, 20, 30, device="cuda")
    ops.muon_step([both[:, 0], both[:, 1]], [g[:2], g[2:]], [mom[:, 1], mom[:, 0]], 0.1)      # (both's and mom's own, crosswise)
    for i in range(4):
        assert torch.equal(both[i % 2, i // 2], want[i]) and torch.equal(mom[i % 2, 1 - i // 2], g[i])
    gaps = torch.ones(2, 2, 20, 30, device="cuda")
    ops.muon_step([gaps[:, 0], gaps[0, 1]], [g[:2], g[2]], [torch.zeros(2, 20, 30, device="cuda"), torch.zeros(20, 30, device="cuda")], 0.1)
    assert torch.equal(gaps[0, 0], want[0]) and torch.equal(gaps[1, 0], want[1]) and torch.equal(gaps[0, 1], want[2])
    assert bool((gaps[1, 1] == 1).all())
    wide = torch.ones(20, 50, device="cuda")
    ops.muon_step([wide[:, :30], wide[4:5, 30:], wide[7:8, 30:]], [g[0], g[1][:1, :20], g[2][:1, :20]],
                  [torch.zeros(20, 30, device="cuda"), torch.zeros(1, 20, device="cuda"), torch.zeros(1, 20, device="cuda")], 0.1)
    assert torch.equal(wide[:, :30], want[0]) and int((wide[:, 30:] != 1).sum(1).gt(0).sum()) == 2
    rows = torch.ones(6, 2, 30, device="cuda")             # stacks of single rows
    ops.muon_step([rows[:, :1], rows[:, 1:]], [g[0][:6, None], g[1][:6, None]], [torch.zeros(6, 1, 30, device="cuda") for _ in range(2)], 0.1)
    assert bool((rows != 1).any(-1).all())


def test_alternating_stacks_that_overlap_are_refused_without_a_gpu():
    lib, C = _lib.lib(), _lib.C
    coef = (C.c_double * 15)(*(COEF * 5))
    base = 1 << 20

    def call(a, b):      # outputs of two stacks of 8 x 8, everything else apart
        arr = (_lib.Matrix * 2)()
        for i, (m, kw) in enumerate(zip(arr, (a, b))):
            d = dict(in_=(4 + i) * base, out=2 * base, momentum=(6 + i) * base, batch=2, rows=8, cols=8, ld_in=8, ld_out=8, ld_momentum=8,
                     in_stride=64, out_stride=128, momentum_stride=64)
            for k, v in {**d, **kw}.items():
                setattr(m, k, v)
        n = lib.dgg_orthogonalize_workspace_bytes(arr, 2)
        return lib.dgg_muon_step(arr, 2, 0.1, 0.9, 1, 0.0, 0, 1.0, coef, 5, 1e-7, 4096, n, None)

    at = 2 * base
    for bad in (({}, dict(out=at + 252)), ({}, dict(out=at + 260)), ({}, dict(out=at + 256, out_stride=129)), ({}, dict(out=at + 256, ld_out=9)),
                ({}, dict(out=at + 256, batch=3, out_stride=64)), ({}, dict(out=at + 128, batch=1)), ({}, dict(out=at + 260, batch=1)),
                (dict(ld_out=16, out_stride=16 * 8), dict(batch=1, rows=1, out=at + 16 * 4 * 3 + 4)),
                (dict(ld_out=16, out_stride=16 * 8), dict(batch=1, rows=1, out=at + 16 * 4 * 3 + 36)),
                (dict(rows=1, out_stride=8), dict(rows=1, out=at + 28, out_stride=16))):
        assert call(*bad) == -1 and b"overlaps" in lib.dgg_last_error(), bad
        assert call(*bad[::-1]) == -1 and b"overlaps" in lib.dgg_last_error(), bad


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((512, 4620), torch.bfloat16), ((24, 257, 771), torch.float32), ((512, 256), torch.float16), ((64, 4108), torch.float32),
                                         ((12, 512), torch.float32)], ids=["wide bf16", "stack f32", "tall f16", "narrow f32", "small f32"])
def test_a_call_repeats_itself_bit_for_bit(shape, dtype):
    """No result depends on the order of workgroups or on what a workspace held before, beside another stream's work."""
    g = torch.randn(shape, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    want = ops.orthogonalize(g)
    side, a = torch.cuda.Stream(), torch.randn(1024, 1024, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    for k in range(20):
        with torch.cuda.stream(side):
            a = a @ a.clamp(-1e-3, 1e-3)
        torch.full((1 << (14 + k % 12),), float("nan"), device="cuda")      # what the allocator hands out next
        assert torch.equal(ops.orthogonalize(g), want), k
    torch.cuda.synchronize()
