"""Thin Python wrappers over the C-ABI (include/dgg.h).  Inputs are torch CUDA tensors (fp32,
contiguous — converted if not); outputs are freshly allocated torch tensors.  No arithmetic happens
here: every function is one or two library calls on the current HIP stream."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_ptr, f32c


def _dev(t):
    if not t.is_cuda:
        raise _lib.DggError("dex_gan_grasp_amd needs CUDA(HIP) tensors; got a %s tensor" % t.device)
    return t.device


# ------------------------------------------------------------------------------------------ A1
def bps_encode(clouds, basis, return_ids=True):
    """clouds (B,N,3) or (N,3), basis (P,3) -> dists (B,P) f32, ids (B,P) int32."""
    dev = _dev(clouds)
    x = f32c(clouds, dev)
    if x.dim() == 2:
        x = x.unsqueeze(0)
    b = f32c(basis, dev)
    B, N, _ = x.shape
    P = b.shape[0]
    dists = torch.empty((B, P), dtype=torch.float32, device=dev)
    ids = torch.empty((B, P), dtype=torch.int32, device=dev) if return_ids else None
    # few clouds of many points (the reference's call shape: one cloud of 15k-73k points) run chunk by chunk on the matrix
    # cores and meet in a workspace; the many-clouds shapes need none (0 bytes)
    nws = int(lib().dgg_bps_workspace_bytes(B, N, P))
    ws = torch.empty((nws,), dtype=torch.uint8, device=dev) if nws > 0 else None
    check(lib().dgg_bps_encode_ws(ptr(x), B, N, ptr(b), P, ptr(dists), ptr(ids), ptr(ws), nws, stream_ptr(dev)),
          "dgg_bps_encode_ws")
    return (dists, ids) if return_ids else dists


# ------------------------------------------------------------------------------------------ GEMM (tests)
def gemm(mode, A, Bm, M, N, K, splits=0, C_out=None, accumulate=False):
    dev = _dev(A)
    out = C_out if C_out is not None else torch.empty((M, N), dtype=torch.float32, device=dev)
    slabs = torch.empty((max(splits, 1) * M * N,), dtype=torch.float32, device=dev) if splits >= 1 else None
    check(lib().dgg_gemm_f32(mode, M, N, K, ptr(A), A.stride(0), ptr(Bm), Bm.stride(0), ptr(out), out.stride(0),
                             splits, ptr(slabs), 1 if accumulate else 0, stream_ptr(dev)), "dgg_gemm_f32")
    return out


# ------------------------------------------------------------------------------------------ networks
def gen_forward(fn, z, bps, train, ws=None):
    dev = fn.device
    z, bps = f32c(z, dev), f32c(bps, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    out = torch.empty((B, fn.ccfg.n_hand_joints + 9), dtype=torch.float32, device=dev)
    check(lib().dgg_gen_forward(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.bn), ptr(ws), ws.numel(), B,
                                _lib.TRAIN if train else 0, ptr(z), ptr(bps), ptr(out), stream_ptr(dev)), "dgg_gen_forward")
    return out


def gen_backward(fn, z, bps, d_heads, train, want_dz=False, want_dbps=False, accumulate=False, ws=None):
    dev = fn.device
    z, bps, d_heads = f32c(z, dev), f32c(bps, dev), f32c(d_heads, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    dz = torch.empty((B, fn.ccfg.latent_d), dtype=torch.float32, device=dev) if want_dz else None
    dbps = torch.empty((B, fn.ccfg.in_bps), dtype=torch.float32, device=dev) if want_dbps else None
    flags = (_lib.TRAIN if train else 0) | (_lib.ACCUM_GRADS if accumulate else 0)
    check(lib().dgg_gen_backward(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.grads), ptr(ws), ws.numel(), B, flags,
                                 ptr(z), ptr(bps), ptr(d_heads), ptr(dz), ptr(dbps), stream_ptr(dev)), "dgg_gen_backward")
    return dz, dbps


def disc_forward(fn, bps, rot9, transl, joint, train, ws=None):
    dev = fn.device
    bps, rot9, transl, joint = f32c(bps, dev), f32c(rot9, dev).reshape(-1, 9), f32c(transl, dev), f32c(joint, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    out = torch.empty((B, 1), dtype=torch.float32, device=dev)
    check(lib().dgg_disc_forward(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.bn), ptr(ws), ws.numel(), B,
                                 _lib.TRAIN if train else 0, ptr(bps), ptr(rot9), ptr(transl), ptr(joint), ptr(out),
                                 stream_ptr(dev)), "dgg_disc_forward")
    return out


def disc_backward(fn, bps, rot9, transl, joint, d_logit, train, need_input=False, skip_param=False, accumulate=False,
                  ws=None):
    dev = fn.device
    bps, rot9, transl, joint = f32c(bps, dev), f32c(rot9, dev).reshape(-1, 9), f32c(transl, dev), f32c(joint, dev)
    d_logit = f32c(d_logit, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    d_pose = torch.empty((B, 12 + fn.ccfg.n_hand_joints), dtype=torch.float32, device=dev) if need_input else None
    flags = (_lib.TRAIN if train else 0) | (_lib.ACCUM_GRADS if accumulate else 0) | \
            (_lib.SKIP_PARAM_GRADS if skip_param else 0) | (_lib.NEED_INPUT_GRADS if need_input else 0)
    check(lib().dgg_disc_backward(C.byref(fn.ccfg), ptr(fn.params), None if skip_param else ptr(fn.grads), ptr(ws),
                                  ws.numel(), B, flags, ptr(bps), ptr(rot9), ptr(transl), ptr(joint), ptr(d_logit),
                                  ptr(d_pose), stream_ptr(dev)), "dgg_disc_backward")
    return d_pose


def eva_forward(fn, bps, rot9, transl, train, drop_keep=None, seed=0, ws=None):
    dev = fn.device
    bps, rot9, transl = f32c(bps, dev), f32c(rot9, dev).reshape(-1, 9), f32c(transl, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    dk = f32c(drop_keep, dev) if drop_keep is not None else None
    out = torch.empty((B, 1), dtype=torch.float32, device=dev)
    check(lib().dgg_eva_forward(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.bn), ptr(ws), ws.numel(), B,
                                _lib.TRAIN if train else 0, ptr(bps), ptr(rot9), ptr(transl), ptr(dk), int(seed),
                                ptr(out), stream_ptr(dev)), "dgg_eva_forward")
    return out


def eva_backward(fn, bps, rot9, transl, d_logit, train, need_input=False, skip_param=False, accumulate=False, ws=None):
    dev = fn.device
    bps, rot9, transl = f32c(bps, dev), f32c(rot9, dev).reshape(-1, 9), f32c(transl, dev)
    d_logit = f32c(d_logit, dev)
    B = bps.shape[0]
    ws = ws if ws is not None else fn.workspace(B)
    d_pose = torch.empty((B, 12), dtype=torch.float32, device=dev) if need_input else None
    flags = (_lib.TRAIN if train else 0) | (_lib.ACCUM_GRADS if accumulate else 0) | \
            (_lib.SKIP_PARAM_GRADS if skip_param else 0) | (_lib.NEED_INPUT_GRADS if need_input else 0)
    check(lib().dgg_eva_backward(C.byref(fn.ccfg), ptr(fn.params), None if skip_param else ptr(fn.grads), ptr(ws),
                                 ws.numel(), B, flags, ptr(bps), ptr(rot9), ptr(transl), ptr(d_logit), ptr(d_pose),
                                 stream_ptr(dev)), "dgg_eva_backward")
    return d_pose


# ------------------------------------------------------------------------------------------ config 5
def _objects_ws(fn, n_obj, n_per):
    key = ("objects", n_obj, n_per)
    ws = fn._ws.get(key)
    if ws is None:
        nb = int(lib().dgg_objects_workspace_bytes(fn.net, C.byref(fn.ccfg), n_obj, n_per))
        if nb < 0:
            raise _lib.DggError("dgg_objects_workspace_bytes: %d" % nb)
        ws = _lib.new_workspace(nb + 4096, fn.device)
        fn._ws[key] = ws
    return ws


def gen_forward_objects(fn, z, bps_obj, n_per):
    """Eval-mode generator over O objects x n_per samples, factorised per object (dgg_gen_forward_objects).
    z (O*n_per, latent), bps_obj (O, 4096) -> heads (O*n_per, nj+9)."""
    dev = fn.device
    z, bps_obj = f32c(z, dev), f32c(bps_obj, dev)
    n_obj = bps_obj.shape[0]
    if z.shape[0] != n_obj * n_per:
        raise _lib.DggError("gen_forward_objects: z has %d rows, expected %d" % (z.shape[0], n_obj * n_per))
    ws = _objects_ws(fn, n_obj, n_per)
    out = torch.empty((n_obj * n_per, fn.ccfg.n_hand_joints + 9), dtype=torch.float32, device=dev)
    check(lib().dgg_gen_forward_objects(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.bn), ptr(ws), ws.numel(), n_obj, n_per,
                                        ptr(z), ptr(bps_obj), ptr(out), stream_ptr(dev)), "dgg_gen_forward_objects")
    return out


def eva_forward_objects(fn, bps_obj, rot9, transl, n_per):
    """Eval-mode evaluator over O objects x n_per samples, factorised per object -> p (O*n_per, 1)."""
    dev = fn.device
    bps_obj, rot9, transl = f32c(bps_obj, dev), f32c(rot9, dev).reshape(-1, 9), f32c(transl, dev)
    n_obj = bps_obj.shape[0]
    if rot9.shape[0] != n_obj * n_per or transl.shape[0] != n_obj * n_per:
        raise _lib.DggError("eva_forward_objects: per-sample inputs need %d rows" % (n_obj * n_per))
    ws = _objects_ws(fn, n_obj, n_per)
    out = torch.empty((n_obj * n_per, 1), dtype=torch.float32, device=dev)
    check(lib().dgg_eva_forward_objects(C.byref(fn.ccfg), ptr(fn.params), ptr(fn.bn), ptr(ws), ws.numel(), n_obj, n_per,
                                        ptr(bps_obj), ptr(rot9), ptr(transl), ptr(out), stream_ptr(dev)),
          "dgg_eva_forward_objects")
    return out


# ------------------------------------------------------------------------------------------ group normalisation
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_ACTS = {"none": _lib.ACT_NONE, "leaky_relu": _lib.ACT_LEAKY_RELU, "silu": _lib.ACT_SILU}


def _stream(dev):
    """The current HIP stream of a tensor's device as an integer (stream_ptr without the Stream object it makes: 2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _launch(dev, call, *args):
    """call(*args) with `dev` the current device: launches go there."""
    if dev.index == torch._C._cuda_getDevice():
        return call(*args)
    with torch.cuda.device(dev):
        return call(*args)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(x):
    """An uninitialised contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _rows(t):
    """t (N, .., C) as (tensor, N, S, C, stride of n, stride of s): the dimensions between the first and the last are one
    axis of S points.  A tensor whose channels do not lie side by side, or whose points are not evenly spaced, is copied."""
    n, c = t.shape[0], t.shape[-1]
    s = t.numel() // (n * c) if n * c else 0
    if t.is_contiguous():
        return t, n, s, c, s * c, c
    mid = [(size, stride) for size, stride in zip(t.shape[1:-1], t.stride()[1:-1]) if size != 1]
    even = all(mid[i][1] == mid[i + 1][0] * mid[i + 1][1] for i in range(len(mid) - 1))
    if (c > 1 and t.stride(-1) != 1) or not even:
        t = t.contiguous()
        return t, n, s, c, s * c, c
    return t, n, s, c, (t.stride(0) if n > 1 else s * c), (mid[-1][1] if mid else c)


def _group_norm_args(who, x, num_groups, weight, bias, act):
    dev = _dev(x)
    if x.dtype not in _DTYPES or x.dim() < 2:
        raise _lib.DggError("%s: x must be (N, .., C) of float32, bfloat16 or float16; got %s %s"
                            % (who, x.dtype, tuple(x.shape)))
    if act not in _ACTS:
        raise _lib.DggError("%s: act must be one of %s; got %r" % (who, sorted(_ACTS), act))
    c = x.shape[-1]
    if c > 1 << 24:
        raise _lib.DggError("%s: %d channels; 2^24 at most" % (who, c))
    if num_groups < 1 or c < 1 or c % num_groups:
        raise _lib.DggError("%s: %d groups do not divide %d channels" % (who, num_groups, c))
    for t in (weight, bias):
        if t is not None and (t.dtype != torch.float32 or t.shape != (c,) or t.device != dev):
            raise _lib.DggError("%s: %s must be a float32 (%d,) tensor on %s; got %s %s on %s"
                                % (who, "weight" if t is weight else "bias", c, dev, t.dtype, tuple(t.shape), t.device))
    return dev, (None if weight is None else weight.contiguous()), (None if bias is None else bias.contiguous())


@functools.lru_cache(maxsize=4096)
def _group_norm_bytes(n, s, c, g, dtype, backward):
    nb = lib().dgg_group_norm_workspace_bytes(n, s, c, g, dtype, backward)
    if nb < 0:
        check(nb, "dgg_group_norm_workspace_bytes")
    return nb


def group_norm_act_forward(x, num_groups, weight=None, bias=None, eps=1e-5, act="leaky_relu", slope=0.2):
    """act(group_norm(x)) over channels-last data: x (N, .., C) float32 / bfloat16 / float16 (a column block of a wider
    product is read in place), num_groups groups of C / num_groups channels, statistics over a sample's points and a group's
    channels; weight / bias float32 (C,) or None; act "none", "leaky_relu" (`slope` for z <= 0) or "silu".
    Returns (y contiguous, of x's shape and type; stats (N, num_groups, 2) float64 = mean and 1 / sqrt(var + eps), which
    group_norm_act_backward takes)."""
    dev, weight, bias = _group_norm_args("group_norm_act_forward", x, num_groups, weight, bias, act)
    y = _like(x)
    stats = x.new_empty((x.shape[0], num_groups, 2), dtype=torch.float64)
    if x.numel() == 0:
        return y, stats.zero_()
    x, n, s, c, sn, ss = _rows(x)
    dt = _DTYPES[x.dtype]
    nb = _group_norm_bytes(n, s, c, num_groups, dt, 0)
    ws = _lib.new_workspace(nb, dev) if nb else None
    check(_launch(dev, lib().dgg_group_norm_act_forward, x.data_ptr(), sn, ss, n, s, c, num_groups, _ptr(weight), _ptr(bias), eps,
                  _ACTS[act], slope, dt, y.data_ptr(), stats.data_ptr(), _ptr(ws), nb, _stream(dev)), "dgg_group_norm_act_forward")
    return y, stats


def group_norm_act_backward(dy, x, num_groups, weight, bias, eps, act, slope, stats, param_grads=True):
    """Gradients of group_norm_act_forward with the same arguments and its `stats`: (dx contiguous, of x's type; dweight,
    dbias float32 (C,), None with param_grads=False)."""
    dev, weight, bias = _group_norm_args("group_norm_act_backward", x, num_groups, weight, bias, act)
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.device != dev:
        raise _lib.DggError("group_norm_act_backward: dy must be like x: %s %s; got %s %s on %s"
                            % (x.dtype, tuple(x.shape), dy.dtype, tuple(dy.shape), dy.device))
    if (stats.shape != (x.shape[0], num_groups, 2) or stats.dtype != torch.float64 or stats.device != dev
            or not stats.is_contiguous()):
        raise _lib.DggError("group_norm_act_backward: stats must be what the forward of the same x returned")
    c = x.shape[-1]
    dx = _like(x)
    dw = db = None
    if param_grads:
        dw = x.new_empty((c,), dtype=torch.float32) if weight is None else torch.empty_like(weight)
        db = x.new_empty((c,), dtype=torch.float32) if bias is None else torch.empty_like(bias)
    if x.numel() == 0:
        return dx, (dw.zero_() if param_grads else None), (db.zero_() if param_grads else None)
    x, n, s, c, sn, ss = _rows(x)
    dy, _, _, _, dsn, dss = _rows(dy)
    dt = _DTYPES[x.dtype]
    nb = _group_norm_bytes(n, s, c, num_groups, dt, 1)
    ws = _lib.new_workspace(nb, dev) if nb else None
    check(_launch(dev, lib().dgg_group_norm_act_backward, dy.data_ptr(), dsn, dss, x.data_ptr(), sn, ss, n, s, c, num_groups,
                  _ptr(weight), _ptr(bias), _ACTS[act], slope, dt, stats.data_ptr(), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), nb,
                  _stream(dev)), "dgg_group_norm_act_backward")
    return dx, dw, db


# ------------------------------------------------------------------------------------------ Newton-Schulz, Muon
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # the quintic whose iterates bring singular values near 1 fast, not exactly to it
_ADJUST = {"spectral": _lib.MUON_SPECTRAL, "match_rms": _lib.MUON_MATCH_RMS}


def _coefficients(who, steps, coefficients):
    """`coefficients`: one (a, b, c) for all steps or a sequence of `steps` of them -> a C array of doubles."""
    rows = [coefficients] * min(steps, 17) if len(coefficients) == 3 and not hasattr(coefficients[0], "__len__") else list(coefficients)
    if not 1 <= steps <= 16 or len(rows) != steps or any(len(r) != 3 for r in rows):
        raise _lib.DggError("%s: 1 to 16 steps and one (a, b, c) for all or for each; got %d, %r" % (who, steps, coefficients))
    return (C.c_double * (3 * steps))(*[float(v) for r in rows for v in r])


def _matrix_rows(t):
    """A matrix or a stack (B, rows, cols) whose rows are contiguous, as (tensor, batch, rows, cols, pitch, stride)."""
    *stack, r, c = t.shape
    b = stack[0] if stack else 1
    if max(r, c) > 1 << 20:
        raise _lib.DggError("matrices of up to 2^20 rows and columns; got %s" % (tuple(t.shape),))
    if t.is_contiguous():
        return t, b, r, c, c, r * c
    if t.stride(-1) != 1 and c > 1 or r > 1 and not c <= t.stride(-2) < 1 << 31:
        t = t.detach().contiguous()
    return t, b, r, c, (t.stride(-2) if r > 1 else c), (t.stride(0) if t.dim() == 3 and b > 1 else r * c)


def _ns_workspace(mats, n, dev):
    nb = lib().dgg_orthogonalize_workspace_bytes(mats, n)
    if nb < 0:
        check(nb, "dgg_orthogonalize_workspace_bytes")
    return _lib.new_workspace(nb, dev), nb


def orthogonalize(grad, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """The orthogonalised form of a matrix (rows, cols), of every matrix of a stack (B, rows, cols), or of each of a list of
    them (one set of launches for the whole list): X_0 = grad / (|grad|_F + eps), then `steps` times
    X <- a X + (b A + c A^2) X with A = X X^T over the shorter side.  float32, bfloat16 or float16 (one type per call);
    returns contiguous tensors of the same shape and type.  No gradient: an optimiser's operator."""
    single = torch.is_tensor(grad)
    grads = [grad] if single else list(grad)
    coef = _coefficients("orthogonalize", steps, coefficients)
    for t in grads:
        dev = _dev(t)
        if t.dtype not in _DTYPES or t.dim() not in (2, 3) or t.dtype != grads[0].dtype or dev != grads[0].device:
            raise _lib.DggError("orthogonalize: matrices (rows, cols) or stacks (B, rows, cols) of one type (float32, bfloat16, "
                                "float16) on one device; got %s %s on %s" % (t.dtype, tuple(t.shape), dev))
    outs = [_like(t.detach()) for t in grads]
    work = [(_matrix_rows(t), o) for t, o in zip(grads, outs) if t.numel()]
    if work:
        dev = grads[0].device
        mats = (_lib.Matrix * len(work))(*[_lib.Matrix(t.data_ptr(), o.data_ptr(), None, b, st, r * c, 0, r, c, ld, c, 0, 0)
                                           for (t, b, r, c, ld, st), o in work])
        ws, nb = _ns_workspace(mats, len(work), dev)
        check(_launch(dev, lib().dgg_orthogonalize, mats, len(work), _DTYPES[grads[0].dtype], coef, steps, eps, ws.data_ptr(), nb,
                      _stream(dev)), "dgg_orthogonalize")
    return outs[0] if single else outs


def muon_step(params, grads, momentum, lr, mu=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NS_COEFFICIENTS,
              eps=1e-7, adjust="spectral", grad_scale=1.0):
    """One Muon step over lists of float32 matrices (or stacks of them), params and momentum in place:
        M <- mu M + grad_scale G;   U = grad_scale G + mu M (nesterov) or M;   W <- (1 - lr weight_decay) W - lr f orthogonalize(U)
    with f = sqrt(max(1, rows / cols)) (adjust="spectral") or 0.2 sqrt(max(rows, cols)) ("match_rms").  A gradient may be
    broadcast; parameters and momenta are written (their version counters advance), so none of them may overlap another tensor
    of the call."""
    who = "muon_step"
    params, grads, momentum = list(params), list(grads), list(momentum)
    if not (len(params) == len(grads) == len(momentum)):
        raise _lib.DggError("%s: %d parameters, %d gradients, %d momenta" % (who, len(params), len(grads), len(momentum)))
    if adjust not in _ADJUST:
        raise _lib.DggError("%s: adjust must be one of %s; got %r" % (who, sorted(_ADJUST), adjust))
    coef = _coefficients(who, steps, coefficients)
    mats, keep, written = [], [], []
    dev = _dev(params[0]) if params else None
    for w, g, m in zip(params, grads, momentum):
        for t in (w, g, m):
            if t.dtype != torch.float32 or t.dim() not in (2, 3) or t.shape != w.shape or t.device != dev:
                raise _lib.DggError("%s: float32 matrices of equal shape on one device are needed; got %s %s on %s"
                                    % (who, t.dtype, tuple(t.shape), t.device))
        if not w.numel():
            continue
        (wt, b, r, c, ldw, sw), (mt, _, _, _, ldm, sm), (gt, _, _, _, ldg, sg) = _matrix_rows(w), _matrix_rows(m), _matrix_rows(g)
        if wt is not w or mt is not m:
            raise _lib.DggError("%s: parameters and momentum are updated in place: their rows must be contiguous and apart" % who)
        keep.append(gt)
        written += (w, m)
        mats.append(_lib.Matrix(gt.data_ptr(), w.data_ptr(), m.data_ptr(), b, sg, sw, sm, r, c, ldg, ldw, ldm, 0))
    if mats:
        n = len(mats)
        mats = (_lib.Matrix * n)(*mats)
        ws, nb = _ns_workspace(mats, n, dev)
        check(_launch(dev, lib().dgg_muon_step, mats, n, lr, mu, int(nesterov), weight_decay, _ADJUST[adjust], grad_scale, coef, steps,
                      eps, ws.data_ptr(), nb, _stream(dev)), "dgg_muon_step")
        # autograd learns that they were written: a graph that still needs their old values raises in its backward pass
        torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])


# ------------------------------------------------------------------------------------------ small ops
def ortho6d_forward(o6):
    dev = _dev(o6)
    o6 = f32c(o6, dev)
    B = o6.shape[0]
    r = torch.empty((B, 9), dtype=torch.float32, device=dev)
    check(lib().dgg_ortho6d_forward(ptr(o6), o6.stride(0), B, ptr(r), stream_ptr(dev)), "dgg_ortho6d_forward")
    return r.view(B, 3, 3)


def ortho6d_backward(o6, d_rot):
    dev = _dev(o6)
    o6, d_rot = f32c(o6, dev), f32c(d_rot, dev).reshape(-1, 9)
    B = o6.shape[0]
    d = torch.empty((B, 6), dtype=torch.float32, device=dev)
    check(lib().dgg_ortho6d_backward(ptr(o6), o6.stride(0), B, ptr(d_rot), ptr(d), 6, stream_ptr(dev)),
          "dgg_ortho6d_backward")
    return d


def bce(p, target, weight=1.0, loss_scale=1.0, want_grad=True):
    """p (B,1) probabilities; target: tensor (B,) / (B,1) of labels or a python float constant.
    Returns (loss 0-d tensor, d_logit (B,1) or None)."""
    dev = _dev(p)
    p = f32c(p, dev)
    B = p.numel()
    labels, const = (f32c(target, dev).reshape(-1), 0.0) if torch.is_tensor(target) else (None, float(target))
    loss = torch.empty((1,), dtype=torch.float32, device=dev)
    dl = torch.empty((B, 1), dtype=torch.float32, device=dev) if want_grad else None
    check(lib().dgg_bce(ptr(p), ptr(labels), const, B, float(weight), float(loss_scale), ptr(loss), ptr(dl),
                        stream_ptr(dev)), "dgg_bce")
    return loss[0], dl


def translate_along_axis(transl, rot9, axis, offset):
    dev = _dev(transl)
    if not transl.is_contiguous() or transl.dtype != torch.float32:
        raise _lib.DggError("translate_along_axis works in place on a contiguous float32 (N, 3) tensor")
    check(lib().dgg_translate_along_axis(ptr(transl), ptr(f32c(rot9, dev)), transl.shape[0], int(axis), float(offset),
                                         stream_ptr(dev)), "dgg_translate_along_axis")
    return transl


def make_hparams(cfg, grad_scale=1.0):
    return _lib.HParams(float(cfg.get("lr_gen", 1e-4)), float(cfg.get("lr_dis", 1e-4)), float(cfg.get("lr", 1e-4)),
                        float(cfg.get("beta1", 0.9)), 0.999, 1e-8, float(cfg.get("weight_decay", 5e-4)),
                        float(cfg.get("bce_weight", 1)), 100.0, 1.0, 10.0, float(grad_scale))
