"""Measured calls of the gated linear recurrence, the layer / RMS norms and the gated RMS norm.

``listed()`` and ``draw()`` give the cases, ``prepare()`` what a user's program has in hand before the call, ``run()`` one
pass -- in plain torch operations in 32 bits, or (``own``) through the public functions of ``mamba_cpu_b200`` --, ``exact()``
the same outputs in 64 bits from the operators' definitions, and ``work()`` the bytes and operations of a pass.

The operators:

* gated linear recurrence: with s_r = sigmoid(decay_gate), s_i = sigmoid(input_gate), per channel A <= 0
      a_t = exp(A s_r),  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) s_i u_t
  the output at step t is h_t. ``seq_idx`` packs sequences into a row: h_{t-1} is dropped where the id changes, and steps
  with a negative id are padding (output 0, state passed on).
* layer norm / RMS norm over the last dimension of the stream s = x + residual, s held in the stream's type;
* gated RMS norm over groups of the last dimension: norm(x * silu(z)) * w, or norm(x) * w * silu(z).
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decoded token of a small model (130M-size d_inner), a handful of users: latency
        dict(name="step 4x1536 bf16", op="step", batch=4, dim=1536, dtype="bf16", state="fp32"),
        # one decoded token at a large serving batch (2.8B-size d_inner)
        dict(name="step 256x5120 bf16", op="step", batch=256, dim=5120, dtype="bf16", state="fp32"),
        # prompt of one user, fp32 weights, the state kept for the decoding that follows
        dict(name="scan prefill 1x1536x1024 fp32", op="scan", batch=1, dim=1536, seqlen=1024, dtype="fp32",
             train=False, packed=False, initial=False),
        # a training step of the 1.4B shape
        dict(name="scan train 8x4096x2048 bf16", op="scan", batch=8, dim=4096, seqlen=2048, dtype="bf16",
             train=True, packed=False, initial=False),
        # packed documents with padded tails, odd sizes, continuing from a state
        dict(name="scan train packed 3x1537x1999 fp16", op="scan", batch=3, dim=1537, seqlen=1999, dtype="fp16",
             train=True, packed=True, initial=True),
        # long-context training of the 2.8B shape
        dict(name="scan train 1x5120x65536 bf16", op="scan", batch=1, dim=5120, seqlen=65536, dtype="bf16",
             train=True, packed=False, initial=False),
        # the block norm of one decoded token, residual stream carried along
        dict(name="rms norm 4x2048 bf16", op="norm", rows=4, dim=2048, dtype="bf16", rms=True, residual="bf16",
             bias=False, pad=0, train=False),
        # the block norm of a 1.4B training step, residual stream in fp32
        dict(name="rms norm train 16384x2048 bf16", op="norm", rows=16384, dim=2048, dtype="bf16", rms=True,
             residual="fp32", bias=False, pad=0, train=True),
        # layer norm in fp32 at odd sizes
        dict(name="layer norm train 4095x769 fp32", op="norm", rows=4095, dim=769, dtype="fp32", rms=False,
             residual="none", bias=True, pad=0, train=True),
        # the norm of the B slice of x_proj's output (dt_rank 128, d_state 16 twice) in training
        dict(name="rms norm train 16384x16 slice bf16", op="norm", rows=16384, dim=16, dtype="bf16", rms=True,
             residual="none", bias=False, pad=144, train=True),
        # the gated norm of one decoded token for a few users
        dict(name="gated norm 8x5120 bf16", op="gate", rows=8, dim=5120, groups=1, dtype="bf16", before=False,
             pad=0, train=False),
        # the gated norm of a training step, z read out of the in-projection's output
        dict(name="gated norm train 16384x4096 bf16", op="gate", rows=16384, dim=4096, groups=1, dtype="bf16",
             before=False, pad=4416, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "norm", "gate"])
    dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    if op == "step":
        return dict(op="step", batch=_log(rng, 1, 256), dim=_log(rng, 64, 5120), dtype=dtype,
                    state=rng.choice(["fp32", dtype]))
    if op == "scan":
        dim, seqlen = _log(rng, 16, 5120), _log(rng, 1, 65536)
        if rng.random() < 0.5 and seqlen >= 16:
            seqlen -= seqlen % 8
        batch = max(1, min(_log(rng, 1, 8), (1 << 27) // (dim * seqlen)))
        return dict(op="scan", batch=batch, dim=dim, seqlen=seqlen, dtype=dtype, train=rng.random() < 0.6,
                    packed=rng.random() < 0.4, initial=rng.random() < 0.4)
    rows = _log(rng, 1, 16384)
    if op == "norm":
        dim = _log(rng, 8, 8192)
        if rng.random() < 0.6 and dim >= 16:
            dim -= dim % 8
        return dict(op="norm", rows=rows, dim=dim, dtype=dtype, rms=rng.random() < 0.5,
                    residual=rng.choice(["none", "fp32", dtype]), bias=rng.random() < 0.5,
                    pad=rng.choice([0, 0, 8, 33]), train=rng.random() < 0.6)
    groups = rng.choice([1, 1, 2, 8])
    dim = groups * max(8, _log(rng, 64, 8192) // groups)
    if rng.random() < 0.6:
        dim -= dim % (8 * groups)
        dim = max(dim, 8 * groups)
    return dict(op="gate", rows=rows, dim=dim, groups=groups, dtype=dtype, before=rng.random() < 0.5,
                pad=rng.choice([0, 0, 16, 2 * dim + 7]), train=rng.random() < 0.6)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=t, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] in ("step", "scan"):
        # decays of 0.9 .. 0.999 a step at a half-open gate, raised to the eighth power at an open one
        s["A"] = 8.0 * torch.log(uniform(0.9, 0.999, case["dim"]))
        if case["op"] == "step":
            shape = (case["batch"], case["dim"])
            s["state"] = normal(*shape, dtype=_DTYPES[case["state"]])
            s["new_state"] = torch.empty_like(s["state"])
            names = ("u", "decay_gate", "input_gate")
        else:
            shape = (case["batch"], case["dim"], case["seqlen"])
            names = ("u", "decay_gate", "input_gate") + (("dy", ) if case["train"] else ())
            if case["initial"]:
                s["initial_state"] = normal(*shape[:2], dtype=torch.float32)
            if case["packed"]:
                # documents of a geometric length around a fifth of the row, and a padded tail
                b, l = case["batch"], case["seqlen"]
                new = torch.rand(b, l, generator=g, device="cuda") < 5.0 / max(l, 8)
                new[:, 0] = False
                ids = torch.cumsum(new, 1)
                used = (uniform(0.8, 1.0, b, 1) * l).ceil()
                s["seq_idx"] = torch.where(torch.arange(l, device="cuda")[None] < used, ids, -1).to(torch.int32)
        for n in names:
            s[n] = normal(*shape)
        grads = ("u", "decay_gate", "input_gate", "A") + (("initial_state", ) if case.get("initial") else ())
    else:
        rows, dim = case["rows"], case["dim"]

        def sliced():  # rows of a wider projection output
            return normal(rows, case["pad"] + dim)[:, case["pad"]:] if case["pad"] else normal(rows, dim)

        if case["op"] == "norm":
            s["x"] = sliced()
            if not case["rms"]:
                s["x"] = s["x"].add_(0.5)
            s["weight"] = 1 + normal(dim, dtype=torch.float32, scale=0.1)
            if case["bias"]:
                s["bias"] = normal(dim, dtype=torch.float32, scale=0.1)
            if case["residual"] != "none":
                s["residual"] = normal(rows, dim, dtype=_DTYPES[case["residual"]], scale=2.0)
            grads = ("x", "weight") + (("bias", ) if case["bias"] else ())
            grads += ("residual", ) if case["residual"] != "none" else ()
            if case["train"]:
                s["dy"] = normal(rows, dim)
                if case["residual"] != "none":
                    s["ds"] = normal(rows, dim, dtype=_DTYPES[case["residual"]])
        else:
            s["x"], s["z"] = normal(rows, dim), sliced()
            s["weight"] = 1 + normal(dim, dtype=torch.float32, scale=0.1)
            grads = ("x", "z", "weight")
            if case["train"]:
                s["dy"] = normal(rows, dim)
    if case.get("train"):
        for n in grads:
            s[n] = s[n].detach().requires_grad_()
        s["grads"] = grads
    return s


_EPS = 1e-5


# ---- the framework's calls ---------------------------------------------------------------------


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-cpu_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mamba_cpu_b200

    return mamba_cpu_b200


def _run_own(s):
    mb, case = _package(), s["case"]
    if case["op"] == "step":
        y = mb.gated_linear_scan_update(s["state"], s["u"], s["decay_gate"], s["input_gate"], s["A"],
                                        out_state=s["new_state"])
        return y, s["new_state"]
    if case["op"] == "scan":
        out = mb.gated_linear_scan_fn(s["u"], s["decay_gate"], s["input_gate"], s["A"], s.get("initial_state"),
                                      s.get("seq_idx"), return_last_state=not case["train"])
        outs, douts = (out, ) if case["train"] else out, (s.get("dy"), )
    elif case["op"] == "norm":
        fn = mb.rms_norm_fn if case["rms"] else mb.layer_norm_fn
        residual = s.get("residual")
        out = fn(s["x"], s["weight"], s.get("bias"), residual, eps=_EPS, prenorm=residual is not None)
        outs, douts = (out if residual is not None else (out, )), (s.get("dy"), s.get("ds"))
    else:
        out = mb.gated_rms_norm_fn(s["x"], s["z"], s["weight"], eps=_EPS, group_size=case["dim"] // case["groups"],
                                   norm_before_gate=case["before"])
        outs, douts = (out, ), (s.get("dy"), )
    if not case["train"]:
        return tuple(outs)
    grads = torch.autograd.grad(outs, [s[n] for n in s["grads"]], douts[:len(outs)])
    return tuple(o.detach() for o in outs), grads


# ---- the plain forms ---------------------------------------------------------------------------


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t along the last dimension (h before the first step is 0): pairs (a, b) are joined over
    distances 1, 2, 4, ..."""
    a, b, n = a.clone(), b.clone(), 1
    while n < a.shape[-1]:
        b[..., n:] += a[..., n:] * b[..., :-n].clone()
        a[..., n:] *= a[..., :-n].clone()
        n *= 2
    return b


def _plain_recurrence(s):
    case = s["case"]
    dtype = s["u"].dtype
    u, r, i = (s[n].detach().float() for n in ("u", "decay_gate", "input_gate"))
    A = s["A"].detach()[:, None] if case["op"] == "scan" else s["A"]
    s_r, s_i = 1 / (1 + torch.exp(-r)), 1 / (1 + torch.exp(-i))
    la = A * s_r
    a = torch.exp(la)
    m = torch.sqrt(-torch.expm1(2 * la))
    b = m * s_i * u
    if case["op"] == "step":
        h = a * s["state"].float() + b
        return h.to(dtype), h.to(s["state"].dtype)
    keep = pad = None
    ak = a
    if case["packed"]:
        ids = s["seq_idx"][:, None, :]
        pad = (ids < 0).expand_as(u)
        keep = torch.ones_like(ids, dtype=torch.bool)
        keep[..., 1:] = (ids[..., 1:] == ids[..., :-1]) | (ids[..., 1:] < 0)
        ak = torch.where(pad, 1.0, torch.where(keep, a, 0.0))
        b = torch.where(pad, 0.0, b)
    h0 = s["initial_state"].detach() if case["initial"] else torch.zeros_like(u[..., 0])
    b = b.clone()
    b[..., 0] += ak[..., 0] * h0
    h = _prefix(ak, b)
    y = h if pad is None else torch.where(pad, 0.0, h)
    if not case["train"]:
        return y.to(dtype), h[..., -1].clone()
    dy = s["dy"].float()
    if pad is not None:
        dy = torch.where(pad, 0.0, dy)
    # g_t = dy_t + a_{t+1} g_{t+1}: the same recurrence from the other end
    back = torch.cat([torch.zeros_like(ak[..., :1]), ak[..., 1:].flip(-1)], -1)
    g = _prefix(back, dy.flip(-1)).flip(-1)
    before = torch.cat([h0[..., None], h[..., :-1]], -1)
    da = g * before if keep is None else torch.where(keep, g * before, 0.0)
    dm = g * s_i * u
    dla = a * da - a * a / m * dm
    du, dr, di = g * m * s_i, dla * A * s_r * (1 - s_r), g * m * u * s_i * (1 - s_i)
    dA = dla * s_r
    if pad is not None:
        du, dr, di, dA = (torch.where(pad, 0.0, v) for v in (du, dr, di, dA))
    grads = (du.to(dtype), dr.to(dtype), di.to(dtype), dA.sum((0, 2)))
    if case["initial"]:
        grads += (ak[..., 0] * g[..., 0], )
    return (y.to(dtype), ), grads


def _plain_norm(s):
    case = s["case"]
    dtype = s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach()
    outs = ()
    if case["residual"] != "none":
        stream = (x + s["residual"].detach().float()).to(s["residual"].dtype)
        outs, x = (stream, ), stream.float()
    xc = x if case["rms"] else x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + _EPS)
    xh = xc * rstd
    y = xh * w
    if case["bias"]:
        y = y + s["bias"].detach()
    outs = (y.to(dtype), ) + outs
    if not case["train"]:
        return outs
    dy = s["dy"].float()
    gw = dy * w
    dx = gw - xh * (gw * xh).mean(-1, keepdim=True)
    if not case["rms"]:
        dx = dx - gw.mean(-1, keepdim=True)
    dx = dx * rstd
    if case["residual"] != "none":
        dx = dx + s["ds"].float()
    grads = (dx.to(dtype), (dy * xh).sum(0))
    if case["bias"]:
        grads += (dy.sum(0), )
    if case["residual"] != "none":
        grads += (dx.to(s["residual"].dtype), )
    return outs, grads


def _plain_gate(s):
    case = s["case"]
    dtype, shape = s["x"].dtype, (case["rows"], case["groups"], case["dim"] // case["groups"])
    x, z = s["x"].detach().float().reshape(shape), s["z"].detach().float().reshape(shape)
    w = s["weight"].detach().reshape(shape[1:])
    sg = 1 / (1 + torch.exp(-z))
    gate = z * sg
    v = x if case["before"] else x * gate
    rstd = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + _EPS)
    vh = v * rstd
    y = vh * w * gate if case["before"] else vh * w
    out = y.to(dtype).reshape(case["rows"], case["dim"])
    if not case["train"]:
        return (out, )
    dy = s["dy"].float().reshape(shape)
    dgate = sg * (1 + z * (1 - sg))
    dn = dy * gate if case["before"] else dy
    gw = dn * w
    dv = rstd * (gw - vh * (gw * vh).mean(-1, keepdim=True))
    if case["before"]:
        dx, dz = dv, dy * vh * w * dgate
    else:
        dx, dz = dv * gate, dv * x * dgate
    flat = (case["rows"], case["dim"])
    return (out, ), (dx.to(dtype).reshape(flat), dz.to(dtype).reshape(flat), (dn * vh).sum(0).reshape(-1))


def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op in ("step", "scan"):
        return _plain_recurrence(s)
    return _plain_norm(s) if op == "norm" else _plain_gate(s)


# ---- 64 bits -----------------------------------------------------------------------------------


def _exact_scan(s):
    """The recurrence step by step, forward and then from the last step back, on (seqlen, batch, dim) arrays."""
    case = s["case"]
    u, r, i = (s[n].detach().double().permute(2, 0, 1).contiguous() for n in ("u", "decay_gate", "input_gate"))
    A = s["A"].detach().double()
    s_r, s_i = torch.sigmoid(r), torch.sigmoid(i)
    a = torch.exp(A * s_r)
    m = torch.sqrt(-torch.expm1(2 * A * s_r))
    b = m * s_i * u
    seqlen = case["seqlen"]
    live = torch.ones(seqlen, case["batch"], 1, dtype=torch.float64, device=u.device)
    joined = live.clone()
    if case["packed"]:
        ids = s["seq_idx"].t()[..., None]
        live = (ids >= 0).double()
        joined[1:] = ((ids[1:] == ids[:-1]) | (ids[1:] < 0)).double()
    carry = torch.where(live > 0, a * joined, torch.ones_like(a))
    b = b * live
    h0 = s["initial_state"].detach().double() if case["initial"] else torch.zeros_like(b[0])
    h = torch.empty_like(b)
    state = h0
    for t in range(seqlen):
        state = torch.addcmul(b[t], carry[t], state, out=h[t])
    y = (h * live).permute(1, 2, 0)
    if not case["train"]:
        return y, h[-1].clone()
    dy = s["dy"].double().permute(2, 0, 1) * live
    g = torch.empty_like(b)
    g[-1] = dy[-1]
    for t in range(seqlen - 2, -1, -1):
        torch.addcmul(dy[t], carry[t + 1], g[t + 1], out=g[t])
    g0 = carry[0] * g[0]
    g = g * live
    prev = torch.cat([h0[None], h[:-1]]) * joined
    slope = g * prev * a - g * s_i * u * a * a / m
    grads = [g * m * s_i, slope * A * s_r * (1 - s_r), g * m * u * s_i * (1 - s_i)]
    grads = [v.permute(1, 2, 0) for v in grads] + [(slope * s_r).sum((0, 1))]
    if case["initial"]:
        grads.append(g0)
    return (y, ), tuple(grads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(s)
    if case["op"] == "step":
        s_r, s_i = torch.sigmoid(s["decay_gate"].double()), torch.sigmoid(s["input_gate"].double())
        la = s["A"].double() * s_r
        h = torch.exp(la) * s["state"].double() + torch.sqrt(-torch.expm1(2 * la)) * s_i * s["u"].double()
        return h, h
    rows, dim = case["rows"], case["dim"]
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    if case["op"] == "norm":
        stream = None
        if case["residual"] != "none":
            stream = (x + s["residual"].detach().double()).to(s["residual"].dtype)
            x = stream.double()
        mean = torch.zeros(rows, 1, dtype=torch.float64, device=x.device) if case["rms"] else x.mean(1, keepdim=True)
        rstd = ((x - mean).square().mean(1, keepdim=True) + _EPS).rsqrt()
        xh = (x - mean) * rstd
        y = torch.addcmul(s["bias"].detach().double(), xh, w) if case["bias"] else xh * w
        outs = (y, ) if stream is None else (y, stream.double())
        if not case["train"]:
            return outs
        dy = s["dy"].double()
        p = dy * w
        dx = rstd * (p - (0 if case["rms"] else p.mean(1, keepdim=True)) - xh * (p * xh).mean(1, keepdim=True))
        if stream is not None:
            dx = dx + s["ds"].double()
        grads = [dx, torch.einsum("rd,rd->d", dy, xh)]
        if case["bias"]:
            grads.append(dy.sum(0))
        if stream is not None:
            grads.append(dx)
        return outs, tuple(grads)
    z = s["z"].detach().double()
    gate = z * torch.sigmoid(z)
    slope = torch.sigmoid(z) * (1 + z - gate)
    n = dim // case["groups"]

    def group_mean(v):
        return v.view(rows, -1, n).mean(2, keepdim=True).expand(-1, -1, n).reshape(rows, dim)

    v = x if case["before"] else x * gate
    rstd = (group_mean(v.square()) + _EPS).rsqrt()
    vh = v * rstd
    y = vh * w * (gate if case["before"] else 1)
    if not case["train"]:
        return (y, )
    dy = s["dy"].double()
    dn = dy * gate if case["before"] else dy
    dv = rstd * (dn * w - vh * group_mean(dn * w * vh))
    dx = dv if case["before"] else dv * gate
    dz = (dy * vh * w if case["before"] else dv * x) * slope
    return (y, ), (dx, dz, torch.einsum("rd,rd->d", dn, vh))


def work(case):
    """Every input read once and every output written once; operations counted from the formulas, a special function as
    one."""
    es = 2 if case["dtype"] != "fp32" else 4
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (4 * es + 2 * (4 if case["state"] == "fp32" else es)) + 4 * case["dim"], "flops": 20 * n}
    if case["op"] == "scan":
        n, rows = case["batch"] * case["dim"] * case["seqlen"], case["batch"] * case["dim"]
        size = n * es * (8 if case["train"] else 4) + 4 * case["dim"] * (2 if case["train"] else 1)
        size += 0 if case["train"] else 4 * rows
        size += 4 * rows * (2 if case["train"] else 1) if case["initial"] else 0
        size += 4 * case["batch"] * case["seqlen"] if case["packed"] else 0
        return {"bytes": size, "flops": n * (60 if case["train"] else 20)}
    n, dim = case["rows"] * case["dim"], case["dim"]
    if case["op"] == "norm":
        rs = {"none": 0, "fp32": 4}.get(case["residual"], es)
        size = n * (2 * es + 2 * rs) * (2 if case["train"] else 1)
        size += 4 * dim * (2 if case["train"] else 1) * (2 if case["bias"] else 1)
        return {"bytes": size, "flops": n * (20 if case["train"] else 6)}
    return {"bytes": n * es * (6 if case["train"] else 3) + 4 * dim * (2 if case["train"] else 1),
            "flops": n * (40 if case["train"] else 12)}
