"""Muon in the framework's own training — FlatNet.muon_step, the engine's and the wrapper's cfg["optimizer"] = "muon", checkpoints —
and networks.GroupNormAct, alone and in a small block that Muon trains.  References and tolerances: test_orthogonalize.py and
test_group_norm.py, from the values that each operator was given; a plain fp32 product of k terms is allowed (k + 1) 2^-24 of the sum
of its terms' absolute values."""
import pytest
import torch

import helpers as H
import test_group_norm as TG
import test_orthogonalize as TO
from dex_gan_grasp_amd import _lib, engine, ops, synth
from dex_gan_grasp_amd.models import networks

CFG = dict(synth.DEFAULT_CFG)
MUON = dict(CFG, optimizer="muon")
U = 2.0 ** -24


def dev_batch(b, seed, with_label=False):
    d = synth.make_batch(b, seed, with_label=with_label)
    last = d["label"] if with_label else d["joint_conf"]
    return tuple(t.float().cuda().contiguous() for t in (d["bps_object"], d["rot_matrix"].reshape(b, 9), d["transl"], last))


def make_engine(cfg):
    fg, fd, fe = (_lib.FlatNet(n, cfg, "cuda") for n in (_lib.NET_GEN, _lib.NET_DISC, _lib.NET_EVA))
    sd = H.gan_sd("wide")
    fg.load_state_dict(sd, "generator.")
    fd.load_state_dict(sd, "discriminator.")
    fe.load_state_dict(H.eva_sd("wide"))
    return engine.TrainEngine(cfg, fg, fd, fe, "cuda")


def copy_of(net, cfg):
    c = _lib.FlatNet(net.net, cfg, "cuda")
    for a in ("params", "grads", "m", "v"):
        getattr(c, a).copy_(getattr(net, a))
    c.step = net.step
    return c


@pytest.mark.parametrize("joints", [12, 7])
@pytest.mark.parametrize("net", [_lib.NET_GEN, _lib.NET_DISC, _lib.NET_EVA])
def test_what_muon_updates(net, joints):
    f = _lib.FlatNet(net, dict(CFG, n_hand_joints=joints), "cpu", with_optim=False)
    names, rest = f.muon_split()
    assert len(names) == (9 if net == _lib.NET_EVA else 6)
    seen = torch.zeros(f.n_params, dtype=torch.int32)
    for e in f.entries:
        if e[0] in names:
            assert e[3] > 1 and e[2] in (256, 512)
            seen[e[1]:e[1] + e[2] * e[3]] += 1
    for lo, hi in rest:
        assert lo % 4 == 0 and lo < hi       # (16-byte loads)
        seen[lo:hi] += 1
    assert bool((seen == 1).all())


def test_refusals_without_a_gpu():
    from dex_gan_grasp_amd.models.dexgangrasp import DexGanGrasp
    with pytest.raises(_lib.DggError):
        engine.optimizer_of({"optimizer": "sgd"})
    assert engine.optimizer_of({}) == engine.optimizer_of(CFG) == "adam"
    with pytest.raises(_lib.DggError):
        DexGanGrasp(dict(CFG, optimizer="sgd"))
    for bad in ((3, 8), (0, 8), (2, 0)):
        with pytest.raises(_lib.DggError):
            networks.GroupNormAct(*bad)
    with pytest.raises(_lib.DggError):
        networks.GroupNormAct(2, 8)(torch.zeros(3, 8))


@pytest.mark.gpu
def test_flat_step_against_the_formulas():
    """The generator: every hidden matrix by the formula in doubles, everything else as one Adam launch over the buffer leaves it."""
    net = _lib.FlatNet(_lib.NET_GEN, CFG, "cuda")
    net.load_state_dict(H.gan_sd("wide"), "generator.")
    names, rest = net.muon_split()
    gen = torch.Generator().manual_seed(3)
    for buf, scale in ((net.grads, 1e-3), (net.m, 1e-3)):
        buf.copy_(torch.randn(net.n_params, generator=gen) * scale)
    net.v.copy_(torch.rand(net.n_params, generator=gen) * 1e-6)
    g = net.views("grads")
    for i, n in enumerate(names):
        g[n].copy_(TO.matrix(*g[n].shape, seed=40 + i))
    net.step = 4
    was, whole = copy_of(net, CFG), copy_of(net, CFG)
    lr, mu, wd, gs = 1e-3, 0.9, 1e-2, 0.5
    net.muon_step(lr, 0.8, 0.99, 1e-7, wd, gs, momentum=mu)
    whole.adam_step(lr, 0.8, 0.99, 1e-7, wd, gs)
    assert net.step == whole.step == 5
    for lo, hi in rest:
        for a in ("params", "m", "v"):
            assert torch.equal(getattr(net, a)[lo:hi], getattr(whole, a)[lo:hi]), (a, lo)
    assert torch.equal(net.grads, was.grads)
    for n in names:
        w, gr, m = (was.views(k)[n].cpu() for k in ("params", "grads", "m"))
        f = 0.2 * max(w.shape) ** 0.5
        rw, rm, tol = TO.muon_reference(w, gr, m, lr, mu, True, wd, f, gs)
        got, gm = net.views("params")[n].cpu().double(), net.views("m")[n].cpu().double()
        assert bool(((gm - rm).abs() <= 3 * U * (m.double().abs() + gs * gr.double().abs() + rm.abs())).all()), n
        err = (got - rw).abs()
        assert float(err.norm()) <= 2 * tol + 4 * U * float(w.norm()), n
        assert bool((err <= 40 * tol / w.numel() ** 0.5 + 4 * U * (w.double().abs() + rw.abs())).all()), n
        assert torch.equal(net.views("v")[n], was.views("v")[n]), n


@pytest.mark.gpu
def test_engine_steps():
    """cgan_step, wgan_step and eva_step leave what their gradients and FlatNet.muon_step give; joint_step on two streams, with
    and without look-ahead, equals the serial steps bit for bit."""
    b = 48
    gan, nxt, eva = dev_batch(b, 1), dev_batch(b, 2), dev_batch(b, 3, with_label=True)
    z = [synth.make_z(b, 7 + i).cuda() for i in range(2)]
    e = make_engine(MUON)
    hp = e._hp()
    kw = (hp.beta1, hp.beta2, hp.eps, hp.weight_decay, hp.grad_scale)

    def follows(net, lr, run):
        before = copy_of(net, MUON)
        run()
        before.grads.copy_(net.grads)
        before.muon_step(lr, *kw)
        assert net.step == before.step
        for a in ("params", "m", "v"):
            assert torch.equal(getattr(net, a), getattr(before, a)), a

    follows(e.E, hp.lr_eva, lambda: e.eva_step(*eva, seed=5))
    follows(e.G, hp.lr_gen, lambda: e.cgan_step(*gan, z[0]))
    alphas = torch.rand(b, 3, device="cuda")
    follows(e.G, hp.lr_gen, lambda: e.wgan_step(*gan, z[0], alphas))
    follows(e.D, hp.lr_dis, lambda: e.cgan_step(*gan, z[0], is_train_gen=False))
    hidden, _ = e.E.muon_split()
    assert all(not e.E.views("v")[n].any() for n in hidden) and all(e.E.views("m")[n].any() for n in hidden)
    with pytest.raises(_lib.DggError):
        e.capture_joint_step(gan, z[0], eva)

    e1, e2, e3 = make_engine(MUON), make_engine(MUON), make_engine(MUON)
    for i, (now, after) in enumerate(((gan, nxt), (nxt, gan))):
        e1.cgan_step(*now, z[i])
        e1.eva_step(*eva, seed=i)
        e2.joint_step(now, z[i], eva, seed=i)
        e3.joint_step(now, z[i], eva, seed=i, next_gan_inputs=after)
    torch.cuda.synchronize()
    for other in (e2, e3):
        for a, c in ((e1.G, other.G), (e1.D, other.D), (e1.E, other.E)):
            assert torch.equal(a.params, c.params) and torch.equal(a.m, c.m) and torch.equal(a.v, c.v) and a.step == c.step
    assert not torch.equal(e1.G.params, make_engine(MUON).G.params)


@pytest.mark.gpu
def test_options():
    cfg = dict(MUON, muon_momentum=0.5, muon_steps=3)
    e = make_engine(cfg)
    eva = dev_batch(32, 3, with_label=True)
    before = copy_of(e.E, cfg)
    e.eva_step(*eva, seed=1)
    before.grads.copy_(e.E.grads)
    hp = e._hp()
    before.muon_step(hp.lr_eva, hp.beta1, hp.beta2, hp.eps, hp.weight_decay, hp.grad_scale, momentum=0.5, steps=3)
    assert torch.equal(e.E.params, before.params)
    e.cfg["muon_steps"] = 0
    with pytest.raises(_lib.DggError):
        e.eva_step(*eva, seed=1)


@pytest.mark.gpu
def test_checkpoints(tmp_path):
    """A run resumed from its checkpoint goes on bit for bit; the state that the other optimiser wrote is not taken over."""
    from dex_gan_grasp_amd.models.dexgangrasp import DexGanGrasp

    def wrapper(optimizer):
        m = DexGanGrasp(dict(CFG, is_train=True, train_ffhevaluator=True, optimizer=optimizer, save_dir=str(tmp_path)))
        m.DexGANGrasp.load_state_dict(H.gan_sd("wide"))
        m.DexEvaluator.load_state_dict(H.eva_sd("wide"))
        return m

    def step(m, i):
        m._z_override = synth.make_z(32, i)
        m._drop_keep = synth.make_dropout_masks(32, 60 + i)
        m.update_dexgangrasp(synth.make_batch(32, i), is_train_gen=True)
        m.update_dexevaluator(synth.make_batch(32, i, with_label=True))

    def nets(m):
        return [x._require_flat() for x in (m.DexGANGrasp.generator, m.DexGANGrasp.discriminator, m.DexEvaluator)]

    def saved(m, name):
        m.save_dexgenerator(name, 1)
        m.save_dexevaluator(name, 1)

    def loaded(optimizer, name):
        m = wrapper(optimizer)
        m.load_dexgenerator(name, str(tmp_path))
        m.load_dexevaluator(name, str(tmp_path))
        return m

    a, adam = wrapper("muon"), wrapper("adam")
    for i in range(2):
        step(a, i)
        step(adam, i)
    saved(a, "muon")
    saved(adam, "adam")
    b = loaded("muon", "muon")
    step(a, 9)
    step(b, 9)
    for x, y in zip(nets(a), nets(b)):
        assert torch.equal(x.params, y.params) and torch.equal(x.m, y.m) and torch.equal(x.v, y.v) and x.step == y.step == 3
    # Muon's state under Adam: all of it starts anew, and a file saved before the first step is Adam's
    c = loaded("adam", "muon")
    for x in nets(c):
        assert x.step == 0 and not x.m.any() and not x.v.any()
    saved(c, "anew")
    d = loaded("adam", "anew")
    step(c, 9)
    step(d, 9)
    for x, y in zip(nets(c), nets(d)):
        assert torch.equal(x.params, y.params) and x.step == 1
    # Adam's state under Muon: the hidden matrices' momentum starts anew, the rest goes on
    e = loaded("muon", "adam")
    for x, y in zip(nets(e), nets(adam)):
        names, rest = x.muon_split()
        assert x.step == 2 and all(not x.views("m")[n].any() and not x.views("v")[n].any() for n in names)
        assert all(torch.equal(x.m[lo:hi], y.m[lo:hi]) and torch.equal(x.v[lo:hi], y.v[lo:hi]) for lo, hi in rest)
    step(e, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ["leaky_relu", "silu", "none"])
def test_group_norm_module(act, dtype):
    n, s, c, g = 5, 37, 48, 6
    x, dy, w, b = TG.data((n, s, c), dtype, 11)
    m = networks.GroupNormAct(g, c, act=act, slope=0.1).cuda()
    with torch.no_grad():
        m.weight.copy_(w)
        m.bias.copy_(b)
    xd = x.cuda().requires_grad_()
    y = m(xd)
    y.backward(dy.cuda())
    want = ops.group_norm_act_forward(xd.detach(), g, m.weight.detach(), m.bias.detach(), 1e-5, act, 0.1)
    grads = ops.group_norm_act_backward(dy.cuda(), xd.detach(), g, m.weight.detach(), m.bias.detach(), 1e-5, act, 0.1, want[1])
    r = TG.reference(x, dy, g, w, b, 1e-5, act, 0.1)
    assert torch.equal(y, want[0]) and y.dtype == dtype
    for got, same in zip((xd.grad, m.weight.grad, m.bias.grad), grads):
        assert torch.equal(got, same)
    TG.close(xd.grad, r["dx"], TG.half_step(dtype, r["dx"]) + r["dx_tol"], "dx")
    # only x or only the parameters want a gradient; x broadcast over the samples; a gradient without memory of its own
    m.zero_grad()
    m(x.cuda()).backward(dy.cuda())
    assert torch.equal(m.bias.grad, grads[2]) and torch.equal(m.weight.grad, grads[1])
    m.requires_grad_(False)
    x2 = x.cuda().requires_grad_()
    m(x2).backward(dy.cuda())
    assert torch.equal(x2.grad, grads[0])
    one = x[:1].cuda().requires_grad_()
    m(one.expand(n, s, c)).sum().backward()
    each = ops.group_norm_act_backward(torch.ones_like(x).cuda(), x[:1].expand(n, s, c).contiguous().cuda(), g, m.weight, m.bias,
                                       1e-5, act, 0.1, ops.group_norm_act_forward(x[:1].expand(n, s, c).cuda(), g, m.weight, m.bias,
                                                                                  1e-5, act, 0.1)[1])[0]
    assert torch.equal(one.grad, each.sum(0, keepdim=True))
    plain = networks.GroupNormAct(g, c, act=act, slope=0.1, affine=False).cuda()
    assert not list(plain.parameters()) and torch.equal(plain(x.cuda()), ops.group_norm_act_forward(x.cuda(), g, None, None, 1e-5, act, 0.1)[0])
    again = networks.GroupNormAct(g, c)
    again.load_state_dict(m.state_dict())
    with pytest.raises(_lib.DggError):
        m(x.cuda()[..., :-1])
    with pytest.raises(RuntimeError):      # once differentiable
        x3 = x.cuda().requires_grad_()
        d, = torch.autograd.grad(m(x3), x3, dy.cuda().requires_grad_(), create_graph=True)
        d.sum().backward()


def block(x, w1, norm, w2):
    h = x @ w1.t()
    y = norm(h)
    return h, y, x + y @ w2.t()


def block_state(seed):
    gen = torch.Generator().manual_seed(seed)
    w1 = (torch.randn(128, 96, generator=gen) / 10).cuda().requires_grad_()
    w2 = (torch.randn(96, 128, generator=gen) / 10).cuda().requires_grad_()
    norm = networks.GroupNormAct(8, 128, device="cuda")
    return w1, w2, norm, [torch.zeros_like(w1), torch.zeros_like(w2)]


@pytest.mark.gpu
def test_a_block_that_muon_trains():
    """Product, group norm with activation, product, residual: every gradient and every update of three steps against doubles, each
    from the values that the operator was given."""
    x = torch.randn(40, 96, generator=torch.Generator().manual_seed(1)).cuda()
    w1, w2, norm, momenta = block_state(2)
    lr, mu, wd = 0.02, 0.95, 0.01
    for k in range(3):
        dout = torch.randn(40, 96, generator=torch.Generator().manual_seed(10 + k)).cuda()
        for p in (w1, w2, norm.weight, norm.bias):
            p.grad = None
        h, y, out = block(x, w1, norm, w2)
        h.retain_grad()
        y.retain_grad()
        out.backward(dout)
        r = TG.reference(h.detach().cpu(), y.grad.cpu(), 8, norm.weight.detach().cpu(), norm.bias.detach().cpu(), 1e-5, "leaky_relu", 0.2)
        TG.close(y.detach(), r["y"], TG.half_step(torch.float32, r["y"]) + (8 + r["z"].abs()) * U * r["y"].abs(), "y")
        TG.close(h.grad, r["dx"], TG.half_step(torch.float32, r["dx"]) + r["dx_tol"], "dh")
        TG.close(norm.weight.grad, r["dw"], r["dw_tol"] + U * r["dw"].abs(), "dweight")
        TG.close(norm.bias.grad, r["db"], r["db_tol"] + U * r["db"].abs(), "dbias")
        for p, left, right in ((w1, h.grad, x), (w2, dout, y.detach())):
            l, rr = left.cpu().double().t(), right.cpu().double()
            TG.close(p.grad, l @ rr, 41 * U * (l.abs() @ rr.abs()), "dW")
        before = [(p.detach().clone().cpu(), m.clone().cpu()) for p, m in zip((w1, w2), momenta)]
        ops.muon_step([w1, w2], [w1.grad, w2.grad], momenta, lr, mu, weight_decay=wd)
        with torch.no_grad():
            for p in (norm.weight, norm.bias):
                p.sub_(lr * p.grad)
        for (w, m), p, pm in zip(before, (w1, w2), momenta):
            f = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
            rw, rm, tol = TO.muon_reference(w, p.grad.cpu(), m, lr, mu, True, wd, f, 1.0)
            assert bool(((pm.cpu().double() - rm).abs() <= 3 * U * (m.double().abs() + p.grad.cpu().double().abs() + rm.abs())).all())
            err = (p.detach().cpu().double() - rw).abs()
            assert float(err.norm()) <= 2 * tol + 4 * U * float(w.norm())
            assert bool((err <= 40 * tol / w.numel() ** 0.5 + 4 * U * (w.double().abs() + rw.abs())).all())


@pytest.mark.gpu
def test_a_captured_block_step():
    """The same step — forward, gradients, Muon — captured once and replayed, against the eager one, replay by replay."""
    def step(x, dout, w1, w2, norm, momenta):
        _, _, out = block(x, w1, norm, w2)
        grads = torch.autograd.grad(out, [w1, w2, norm.weight, norm.bias], dout)
        ops.muon_step([w1, w2], grads[:2], momenta, 0.02, weight_decay=0.01)
        with torch.no_grad():
            norm.weight.sub_(0.02 * grads[2])
            norm.bias.sub_(0.02 * grads[3])

    x, dout = torch.zeros(40, 96, device="cuda"), torch.zeros(40, 96, device="cuda")
    mine, eager = block_state(2), block_state(2)
    warm = block_state(5)
    step(x + 1, dout + 1, *warm)          # library handles come into being outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, dout, *mine)
    for k in range(4):
        gen = torch.Generator().manual_seed(20 + k)
        x.copy_(torch.randn(40, 96, generator=gen))
        dout.copy_(torch.randn(40, 96, generator=gen))
        graph.replay()
        step(x, dout, *eager)
        torch.cuda.synchronize()
        for a, b in zip([mine[0], mine[1], mine[2].weight, mine[2].bias] + mine[3], [eager[0], eager[1], eager[2].weight, eager[2].bias] + eager[3]):
            assert torch.equal(a, b), k


@pytest.mark.gpu
def test_calls_from_several_threads_at_once():
    """Each thread on a stream of its own, all routes of both operators: every result as on one stream."""
    import threading
    shapes = [(20, 30), (64, 190), (20, 900), (64, 1300), (100, 200), (200, 300)]
    gs = [TO.matrix(*s, seed=i).cuda() for i, s in enumerate(shapes)]
    xs = [(TG.data((n, s, c), torch.float32, 3)[0].cuda(), g) for n, s, c, g in ((64, 1, 512, 32), (4, 300, 64, 8), (2, 9000, 4, 1))]
    want = [ops.orthogonalize(g) for g in gs], [ops.group_norm_act_forward(x, g) for x, g in xs]
    back = [ops.group_norm_act_backward(x, x, g, None, None, 1e-5, "leaky_relu", 0.2, y[1]) for (x, g), y in zip(xs, want[1])]
    torch.cuda.synchronize()
    bad = []

    def run(turn):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for k in range(6):
                    order = [(turn + k + i) % len(gs) for i in range(len(gs))]
                    got = {i: ops.orthogonalize(gs[i]) for i in order}
                    for (x, g), (y, st), b in zip(xs, want[1], back):
                        gy, gst = ops.group_norm_act_forward(x, g)
                        gb = ops.group_norm_act_backward(x, x, g, None, None, 1e-5, "leaky_relu", 0.2, gst)
                        if not (torch.equal(gy, y) and torch.equal(gst, st) and all(torch.equal(p, q) for p, q in zip(gb, b))):
                            bad.append(("group norm", turn, k, tuple(x.shape)))
                    bad.extend(("orthogonalize", turn, k, shapes[i]) for i, o in got.items() if not torch.equal(o, want[0][i]))
        except Exception as e:
            bad.append((turn, repr(e)))

    threads = [threading.Thread(target=run, args=(t,)) for t in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, bad[:5]
