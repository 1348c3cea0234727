"""CUDA layer norm, RMS norm and gated RMS norm, forward and backward, against float64.

Tolerances: half a step of the output's type plus the float32 kernel's error in units of 2^-24 of the
largest value. A row's sums add at most 16 terms in a thread, 5 in a warp and 32 over warps, so the
statistics are off by at most 53 units, half of that in the root; the factors around them and the
gate (whose fast exponential is off by up to 2 + 1.2 |z| units in the last place, |z| < 6) add less
than 40. So: 96 for outputs, twice that for gradients, whose terms carry two statistics. Sums over
rows: one more unit per row, of the sum of the terms' sizes."""

import threading

import pytest
import torch

import block_oracles as bo
import mamba_cpu_b200 as mb
from mamba_cpu_b200 import _lib

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rand(*shape, dtype=F32, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def place(t, pad):
    """t on the GPU; with `pad` as columns of a wider buffer of NaN, that many elements behind the start of its rows."""
    if not pad:
        return t.cuda()
    wide = torch.full((t.shape[0], pad + t.shape[1] + 2), float("nan"), dtype=t.dtype, device="cuda")
    return wide[:, pad:pad + t.shape[1]].copy_(t)


def run_norm(fn, t, prenorm, train=True, pad=0):
    c = {k: None if v is None else place(v, pad) if k in ("x", "res") else v.cuda() for k, v in t.items()}
    leaves = {k: c[k].detach().requires_grad_(train) for k in ("x", "w", "b", "res") if c.get(k) is not None}
    out = fn(leaves["x"], leaves.get("w"), leaves.get("b"), leaves.get("res"), prenorm=prenorm)
    outs = out if prenorm else (out,)
    if not train:
        return outs, None
    grads = torch.autograd.grad(outs, list(leaves.values()), (c["dy"], c["ds"])[:len(outs)])
    return outs, dict(zip(leaves, grads))


def check_norm(rms, rows, n, dtype, res=None, bias=True, weight=F32, prenorm=True, seed=0, train=True, pad=0):
    """`res`: the residual's dtype or None."""
    prenorm = prenorm and res is not None
    t = dict(x=rand(rows, n, dtype=dtype, seed=seed, shift=0.3), dy=rand(rows, n, dtype=dtype, seed=seed + 1),
             w=None if weight is None else rand(n, dtype=weight, seed=seed + 2, scale=0.2, shift=1.0),
             b=rand(n, dtype=weight or F32, seed=seed + 3) if bias else None,
             res=None if res is None else rand(rows, n, dtype=res, seed=seed + 4, scale=1.5),
             ds=None if res is None else rand(rows, n, dtype=res, seed=seed + 5))
    outs, grads = run_norm(mb.rms_norm_fn if rms else mb.layer_norm_fn, t, prenorm, train, pad)
    want = bo.norm(t["x"], t["w"], t["b"], t["res"], res or F32, rms=rms, dy=t["dy"], ds=t["ds"] if prenorm else None)
    assert outs[0].dtype == dtype
    bo.check(outs[0], want["out"], dtype, 96, name="out")
    if prenorm:
        assert outs[1].dtype == res
        bo.check(outs[1], want["s"], res, 0, name="sum")
    if not train:
        return
    # a row of one column (and, in layer norm, of two) is normalised to a constant: its gradient is what is left of
    # terms of the size of dy rstd
    big = float((abs(bo.f64(t["dy"])) * want["rstd"]).max()) * 2 + float(abs(want["dx"]).max())
    bo.check(grads["x"], want["dx"], dtype, 192, scale=big, name="dx")
    if weight is not None:
        assert grads["w"].dtype == weight
        bo.check(grads["w"], want["dw"], weight, 192 + rows, scale=want["dw_abs"], name="dw")
    if bias:
        bo.check(grads["b"], want["db"], weight or F32, 192 + rows, scale=want["db_abs"], name="db")
    if res is not None:
        assert grads["res"].dtype == res
        bo.check(grads["res"], want["dx"], res, 192, scale=big, name="dres")


@pytest.mark.parametrize("n", [1, 2, 3, 8, 16, 17, 31, 64, 100, 255, 256, 511, 512, 513, 520, 769, 1024, 2048, 2050,
                               4100, 5120, 8192])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_widths(n, rms, dtype):
    check_norm(rms, 5, n, dtype, seed=n)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 1000, 20000])
@pytest.mark.parametrize("n", [16, 24, 640])
def test_rows(rows, n):
    check_norm(True, rows, n, BF16, res=BF16, bias=False, seed=rows)


@pytest.mark.parametrize("n", [12000, 16383, 16384])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_widest(n, dtype):
    check_norm(False, 3, n, dtype, res=F32, seed=1)


@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("n", [48, 333, 1536])
@pytest.mark.parametrize("prenorm", [False, True])
def test_residual(dtype, res, rms, n, prenorm):
    check_norm(rms, 70, n, dtype, res=res, prenorm=prenorm, seed=n)


@pytest.mark.parametrize("rows,n", [(5001, 256), (3001, 264), (1500, 512), (700, 768), (701, 2048), (400, 4096), (333, 5120)])
@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rms", [False, True])
def test_residual_rows(rows, n, dtype, res, rms):
    """Several rows to a team, so that rows are copied one or two ahead, at the widths of every layout."""
    check_norm(rms, rows, n, dtype, res=res, seed=n)


@pytest.mark.parametrize("pad", [1, 2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("rows,n", [(1, 8), (40, 9), (700, 40), (2600, 257), (400, 2048), (350, 2051), (170, 5119), (20, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shifted_rows(rows, n, dtype, pad):
    """Inputs at every offset of a wider buffer, whose rows are aligned in another way than the results'."""
    check_norm(pad % 2 == 0, rows, n, dtype, res=None if pad % 3 else F32, seed=n, pad=pad)
    check_gated(rows, n, None, dtype, pad % 2 == 1, seed=n, pad=pad)


@pytest.mark.parametrize("weight", [None, F32, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_weight_types(weight, bias):
    check_norm(False, 33, 200, BF16, res=F32, bias=bias, weight=weight)
    check_norm(True, 33, 1200, BF16, bias=bias, weight=weight)


@pytest.mark.parametrize("rms", [False, True])
def test_inference(rms):
    for n in (40, 41, 2048):
        check_norm(rms, 9, n, BF16, res=F32, train=False)
        check_norm(rms, 9, n, F32, train=False)


def check_gated(rows, n, group, dtype, before, weight=F32, seed=0, train=True, pad=0):
    x, z = rand(rows, n, dtype=dtype, seed=seed), rand(rows, n, dtype=dtype, seed=seed + 1)
    dy = rand(rows, n, dtype=dtype, seed=seed + 2)
    w = None if weight is None else rand(n, dtype=weight, seed=seed + 3, scale=0.2, shift=1.0)
    leaves = [place(x, pad), place(z, 0 if pad == 3 else pad)] + ([] if w is None else [w.cuda()])
    leaves = [t.requires_grad_(train) for t in leaves]
    y = mb.gated_rms_norm_fn(leaves[0], leaves[1], leaves[2] if w is not None else None, group_size=group,
                             norm_before_gate=before)
    want = bo.gated(x, z, w, group=group, before=before, dy=dy)
    bo.check(y, want["out"], dtype, 96, name="out")
    if not train:
        return
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    bo.check(grads[0], want["dx"], dtype, 192, name="dx")
    bo.check(grads[1], want["dz"], dtype, 192, name="dz")
    if w is not None:
        assert grads[2].dtype == weight
        bo.check(grads[2], want["dw"], weight, 192 + rows, scale=want["dw_abs"], name="dw")


@pytest.mark.parametrize("n,group", [(8, None), (24, None), (33, None), (33, 11), (64, 16), (520, 260), (1536, None),
                                     (1538, None), (4096, 512), (5120, 640), (2047, None), (4096, 4096)])
@pytest.mark.parametrize("before", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_gated(n, group, before, dtype):
    check_gated(37, n, group, dtype, before, seed=n)


@pytest.mark.parametrize("rows", [1, 2, 4000])
@pytest.mark.parametrize("before", [False, True])
def test_gated_rows(rows, before):
    check_gated(rows, 96, 48, BF16, before)
    check_gated(rows, 768, None, F32, before, weight=None)
    check_gated(rows, 768, 384, BF16, before, weight=BF16)
    check_gated(rows, 768, 384, BF16, before, train=False)


def test_gated_widest():
    check_gated(2, 32768, 16384, BF16, False)
    check_gated(2, 16384, None, F32, True)
    check_gated(2, 16383, None, F16, False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype):
    """Leading dimensions, slices, odd addresses, broadcasts: results and gradients of the dense call."""
    g, b, n = 4, 6, 96
    x, z = rand(g, b, n, dtype=dtype).cuda(), rand(g, b, n, dtype=dtype, seed=1).cuda()
    w, dy = rand(n, seed=2).cuda(), rand(g, b, n, dtype=dtype, seed=3).cuda()

    def within(t, before, after):
        big = torch.full(t.shape[:-1] + (before + n + after,), float("nan"), dtype=t.dtype, device="cuda")
        big[..., before:before + n] = t
        return big[..., before:before + n]

    def calls(x, z):
        xl, zl, wl = (t.detach().requires_grad_() for t in (x, z, w))
        y, s = mb.layer_norm_fn(xl, wl, residual=zl, prenorm=True)
        a = (y, s) + torch.autograd.grad((y, s), (xl, zl, wl), (dy, dy))
        y = mb.gated_rms_norm_fn(xl, zl, wl, group_size=32)
        return a + (y,) + torch.autograd.grad(y, (xl, zl, wl), dy)

    ref = calls(x, z)
    swap = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    last = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for f in (lambda t: within(t, 8, 16), lambda t: within(t, 0, 40), lambda t: within(t, 3, 2), swap, last):
        for got in (calls(f(x), f(z)), calls(x, f(z)), calls(f(x), z)):
            for a, r in zip(got, ref):
                # an unaligned row is summed in another order: 2 units of the sums' 53
                torch.testing.assert_close(a, r, rtol=1e-2 if dtype == BF16 else 2e-5, atol=1e-2 if dtype == BF16 else 2e-5)
    one = x[:1, :1].expand(g, b, n)
    y = mb.rms_norm_fn(one, w)
    assert torch.equal(y, mb.rms_norm_fn(one.contiguous(), w))
    leaf = x[:1].clone().requires_grad_()
    gl, = torch.autograd.grad(mb.rms_norm_fn(leaf.expand(g, b, n), w), leaf, dy)
    assert gl.shape == leaf.shape
    vec = x[0, 0].clone()
    assert torch.equal(mb.rms_norm_fn(vec, w), mb.rms_norm_fn(vec[None], w)[0])


def test_rows_do_not_touch():
    """NaN or infinity in one row stays there; rows of zeros give the bias, and finite gradients."""
    x = rand(50, 256, seed=4).cuda()
    w, b = rand(256, seed=5).cuda(), rand(256, seed=6).cuda()
    ref = mb.layer_norm_fn(x, w, b)
    y = x.clone()
    y[7], y[9, 3] = float("nan"), float("inf")
    y[11] = 0
    got = mb.layer_norm_fn(y, w, b)
    others = [k for k in range(50) if k not in (7, 9, 11)]
    assert torch.equal(got[others], ref[others]) and torch.isnan(got[[7, 9]]).all() and torch.equal(got[11], b)
    zero = torch.zeros(3, 256, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(mb.rms_norm_fn(zero, w), zero, x[:3])
    torch.testing.assert_close(g, x[:3] * w / 1e-5 ** 0.5, rtol=1e-5, atol=0)
    eps0 = mb.rms_norm_fn(x, w, eps=0.0)
    assert torch.isfinite(eps0).all()
    leaf = w.clone().requires_grad_()
    gw, = torch.autograd.grad(mb.rms_norm_fn(x[:3], leaf, eps=0.0), leaf, x[:3])  # idle teams have no row
    assert torch.isfinite(gw).all()


def test_large_mean():
    """Layer norm of rows far from zero: the mean is taken off before the squares."""
    x = rand(20, 1000, seed=8, shift=300.0)
    y = mb.layer_norm_fn(x.cuda(), None)
    want = bo.norm(x, rms=False)
    # the mean's own rounding, 53 units of 300, moves a row by that much
    bo.check(y, want["out"], F32, 96 + 2 * 53 * 300, scale=1.0, name="out")


def test_16bit_extremes():
    """fp16 rows near the type's end: squares are float32 sums, and the stream rounds as the type does."""
    x = rand(8, 512, dtype=F16, seed=9) * 10000
    check = mb.rms_norm_fn(x.cuda(), None)
    bo.check(check, bo.norm(x, rms=True)["out"], F16, 96, name="out")
    a = torch.full((2, 64), 60000.0, dtype=F16).cuda()
    y, s = mb.rms_norm_fn(a, None, residual=a, prenorm=True)
    assert torch.isinf(s).all() and torch.isnan(y).all()
    y, s = mb.rms_norm_fn(a, None, residual=a, prenorm=True, residual_in_fp32=True)
    assert s.dtype == F32 and (s == 120000.0).all() and (y == 1).all()


@pytest.mark.parametrize("shape", [(0, 8), (3, 0), (0, 0), (2, 0, 16)])
def test_empty(shape):
    n = shape[-1]
    x, w = torch.zeros(shape, device="cuda", requires_grad=True), torch.ones(n, device="cuda", requires_grad=True)
    for y in (mb.rms_norm_fn(x, w), mb.layer_norm_fn(x, w, w), mb.gated_rms_norm_fn(x, x, w)):
        assert y.shape == shape
        gx, gw = torch.autograd.grad(y, (x, w), torch.zeros(shape, device="cuda"))
        assert gx.shape == shape and gw.shape == (n,) and not gw.any()


def test_other_types_and_unused_outputs():
    x = rand(6, 40).cuda()
    w = rand(40, seed=1).cuda()
    y = mb.rms_norm_fn(x.double(), w.double())
    assert y.dtype == torch.float64 and torch.equal(y.float(), mb.rms_norm_fn(x, w))
    xb = x.to(BF16).requires_grad_()
    res = x.to(F16).requires_grad_()
    y, s = mb.rms_norm_fn(xb, w.to(F16), residual=res, prenorm=True)
    assert s.dtype == F32 and y.dtype == BF16
    gx, gr = torch.autograd.grad(s, (xb, res), torch.ones_like(s), retain_graph=True)  # y has no gradient
    assert gx.dtype == BF16 and gr.dtype == F16 and (gx == 1).all() and (gr == 1).all()
    gx, = torch.autograd.grad(y, xb, torch.ones_like(y))  # s has none
    assert torch.isfinite(gx).all()
    y, s = mb.rms_norm_fn(xb, w, prenorm=True)
    assert s is xb
    y, s = mb.rms_norm_fn(xb, w, prenorm=True, residual_in_fp32=True)
    assert s.dtype == F32
    z = x.to(BF16)
    assert torch.equal(mb.gated_rms_norm_fn(x, z, w), mb.gated_rms_norm_fn(x, z.float(), w))
    same = x.clone().requires_grad_()
    y, s = mb.rms_norm_fn(same, w, residual=same, prenorm=True)  # one tensor as both
    g, = torch.autograd.grad((y, s), same, (x, x))
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    y2, s2 = mb.rms_norm_fn(a, w, residual=b, prenorm=True)
    ga, gb = torch.autograd.grad((y2, s2), (a, b), (x, x))
    assert torch.equal(g, ga + gb)


def _training_call(seed, n=1024):
    x, r, z = (rand(300, n, dtype=BF16, seed=seed + k).cuda().requires_grad_() for k in range(3))
    w = rand(n, seed=seed + 3).cuda().requires_grad_()
    dy = rand(300, n, dtype=BF16, seed=seed + 4).cuda()

    def call():
        y, s = mb.rms_norm_fn(x, w, residual=r, prenorm=True)
        o = mb.gated_rms_norm_fn(y, z, w, group_size=256)
        return (y, s, o) + torch.autograd.grad((o, s), (x, r, z, w), (dy, dy))

    return call, (x, dy)


@pytest.mark.parametrize("n", [1024, 8192])
def test_captured_and_replayed(n):
    made = [_training_call(10 * k, n) for k in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c, _ in made:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c, _ in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    for turn in range(2):
        for _, (x, dy) in made:
            with torch.no_grad():
                x.mul_(-0.5)
                dy.add_(0.25)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (c, _), o in zip(made, outs):
            assert all(torch.equal(a, b) for a, b in zip(c(), o))


def test_streams_and_threads():
    calls = [_training_call(10 * k)[0] for k in range(4)]
    ref = [c() for c in calls]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[k] = calls[k]()
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for r, g in zip(ref, got):
        assert all(torch.equal(a, b) for a, b in zip(r, g))


def test_threads_with_different_widths():
    """Calls of one kernel at widths that ask for different amounts of shared memory, from two threads at once through
    the C ABI (which leaves the interpreter's lock alone): every one is launched with what it asked for."""
    def forward(n):
        x, z, w = (rand(r, n, dtype=BF16, seed=r + k).cuda() for k, r in enumerate((4, 4, 1)))
        out = torch.empty_like(x)
        p = _lib.NormParams(x=x.data_ptr(), z=z.data_ptr(), weight=w.data_ptr(), out=out.data_ptr(), rows=4, dim=n,
                            group_size=n, eps=1e-5, io_dtype=_lib.BF16, residual_dtype=_lib.BF16, weight_dtype=_lib.BF16,
                            rms=1, gate=_lib.GATE_BEFORE_NORM)
        return lambda s: _lib.lib.mb200_norm_fwd(p, s), out, mb.gated_rms_norm_fn(x, z, w[0]), (x, z, w)

    def backward(n):
        dy, s, w = rand(4, n, dtype=BF16).cuda(), rand(4, n, seed=1).cuda(), rand(n, seed=2).cuda()
        dx, dw = torch.empty_like(dy), torch.empty_like(w)
        f = _lib.NormParams(x=s.data_ptr(), residual=s.data_ptr(), weight=w.data_ptr(), rows=4, dim=n, group_size=n,
                            eps=1e-5, io_dtype=_lib.BF16, rms=1)
        p = _lib.NormBwdParams(fwd=f, dout=dy.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr())
        ref = torch.ops.mamba_b200.norm_bwd(dy, None, s, None, w, F32, None, 1e-5, n, True, 0, False)[0]
        size = _lib.lib.mb200_norm_bwd_workspace_size(p)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        return lambda st: _lib.lib.mb200_norm_bwd(p, ws.data_ptr(), size, st), dx, ref, (dy, s, w, dw, ws)

    for make, widths in ((forward, (4096, 5120)), (backward, (512, 1024))):
        cases = [make(n) for n in widths]
        torch.cuda.synchronize()
        refused = [0, 0]

        def work(k):
            stream = torch.cuda.Stream()
            for _ in range(20000):
                refused[k] += cases[k][0](stream.cuda_stream) != 0
            stream.synchronize()

        threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert refused == [0, 0], f"{make.__name__}: launches refused {refused}"
        assert all(torch.equal(out, ref) for _, out, ref, _ in cases)


@pytest.mark.parametrize("rows", [3, 700])
def test_frozen_weight(rows):
    """A weight that asks for no gradient gets no sums over the rows; the other gradients are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Sums(TorchDispatchMode):  # sizes of dweight and dbias of the backward calls
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func is torch.ops.mamba_b200.norm_bwd.default:
                self.seen.append((out[3].numel(), out[4].numel()))
            return out

    n = 200
    x, z, dy = (rand(rows, n, dtype=BF16, seed=k).cuda() for k in range(3))
    w, b = rand(n, seed=3).cuda(), rand(n, seed=4).cuda()
    calls = [(lambda x, w, b: mb.layer_norm_fn(x, w, b, residual=z), True), (lambda x, w, b: mb.rms_norm_fn(x, w), False),
             (lambda x, w, b: mb.gated_rms_norm_fn(x, z, w), False)]
    for call, biased in calls:
        all_of = [t.clone().requires_grad_() for t in ((x, w, b) if biased else (x, w))]
        want = torch.autograd.grad(call(*(all_of + [b])[:3]), all_of, dy)
        for wants_b in ((False, True) if biased else (False,)):
            xl, bl = x.clone().requires_grad_(), b.clone().requires_grad_(wants_b)
            y = call(xl, w, bl)
            with Sums() as mode:
                mode.seen = []
                got = torch.autograd.grad(y, [xl, bl] if wants_b else [xl], dy)
            assert mode.seen == [(0, n if wants_b else 0)]
            assert torch.equal(got[0], want[0]) and (not wants_b or torch.equal(got[1], want[2]))


def test_first_order_only():
    """Gradients that are asked to be differentiable come, and raise when they are differentiated."""
    x, w, dy = rand(5, 40).cuda().requires_grad_(), rand(40, seed=1).cuda(), rand(5, 40, seed=2).cuda()
    for f in (lambda t: mb.layer_norm_fn(t, w), lambda t: mb.gated_rms_norm_fn(t, dy, w)):
        g, = torch.autograd.grad(f(x), x, dy, create_graph=True)
        assert torch.equal(g, torch.autograd.grad(f(x), x, dy)[0])
        if g.requires_grad:
            with pytest.raises(RuntimeError):
                torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("call", ["layer", "rms", "gated"])
def test_second_backward_raises(call):
    """A gradient that was asked to be differentiable says so, and differentiating it raises, whichever input it is of."""
    x, w, b, z, dy = (t.cuda() for t in (rand(5, 40), rand(40, seed=1), rand(40, seed=2), rand(5, 40, seed=3), rand(5, 40, seed=4)))
    leaves = [t.requires_grad_() for t in ((x, z, w) if call == "gated" else (x, z, w, b))]
    if call == "gated":
        y = mb.gated_rms_norm_fn(x, z, w)
    else:
        y = (mb.layer_norm_fn if call == "layer" else mb.rms_norm_fn)(x, w, b, z)
    grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for g in grads:
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="norm_bwd is not implemented"):
            torch.autograd.grad(g.sum(), x, retain_graph=True)


def test_compiled():
    """Traced and run by torch.compile's eager backend, gradients included."""
    x, r, z = (rand(6, 64, seed=k).cuda().requires_grad_() for k in range(3))
    w, dy = rand(64, seed=3).cuda().requires_grad_(), rand(6, 64, seed=4).cuda()

    def f(x, r, z, w):
        y, s = mb.rms_norm_fn(x, w, residual=r, prenorm=True)
        return mb.gated_rms_norm_fn(y, z, w, group_size=16) * 2, s

    got, want = torch.compile(f, backend="aot_eager", fullgraph=True)(x, r, z, w), f(x, r, z, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ga, gb = (torch.autograd.grad(o, (x, r, z, w), (dy, dy)) for o in (got, want))
    assert all(torch.equal(a, b) for a, b in zip(ga, gb))


@pytest.mark.parametrize("offset", range(1, 8))
@pytest.mark.parametrize("n", [1, 3, 7, 9])
def test_narrow_rows_at_odd_addresses(n, offset):
    """Rows of a few columns that begin anywhere in a buffer, up against its ends: nothing outside is read into the
    sums, and nothing outside is written."""
    for dtype in (F32, BF16):
        rows = 41
        buf = torch.full((rows * n + offset,), float("nan"), dtype=dtype, device="cuda")
        x = rand(rows, n, dtype=dtype, seed=n)
        buf[offset:] = x.cuda().flatten()
        view = buf[offset:].view(rows, n).requires_grad_()
        w = rand(n, seed=2).cuda().requires_grad_()
        dy = rand(rows, n, dtype=dtype, seed=3)
        y = mb.rms_norm_fn(view, w)
        gx, gw = torch.autograd.grad(y, (view, w), dy.cuda())
        want = bo.norm(x, w.detach(), rms=True, dy=dy)
        bo.check(y, want["out"], dtype, 96, name="out")
        big = float((abs(bo.f64(dy)) * want["rstd"]).max()) * 2 * float(abs(bo.f64(w)).max())
        bo.check(gx, want["dx"], dtype, 192, scale=big, name="dx")
        bo.check(gw, want["dw"], F32, 192 + rows, scale=want["dw_abs"], name="dw")


@pytest.mark.slow
def test_offsets_past_32_bits():
    """More than 2^31 elements a tensor: the last rows are those of a call on them alone."""
    rows, n = 270000, 8192
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.empty(rows, n, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(2))
    w = torch.randn(n, device="cuda", generator=g)
    leaf = x.requires_grad_()
    y = mb.rms_norm_fn(leaf, w)
    gx, = torch.autograd.grad(y, leaf, dy)
    tail = x.detach()[-3:].clone().requires_grad_()
    y2 = mb.rms_norm_fn(tail, w)
    assert torch.equal(y[-3:], y2) and torch.equal(gx[-3:], torch.autograd.grad(y2, tail, dy[-3:])[0])


def test_opcheck():
    x, z, w = (t.cuda() for t in (rand(5, 32, dtype=BF16), rand(5, 32, dtype=BF16, seed=1), rand(32, seed=2)))
    r = rand(5, 32, seed=3).cuda()
    ops, utils = torch.ops.mamba_b200, ("test_schema", "test_faketensor")
    for args in ((x, r, None, w, w, 1e-5, 32, False, 0, True), (x, None, z, w, None, 1e-5, 8, True, 2, False)):
        torch.library.opcheck(ops.norm_fwd.default, args, test_utils=utils)
    for args in ((x, r, r, None, w, F32, F32, 1e-5, 32, False, 0, True), (x, None, x, z, w, None, None, 1e-5, 8, True, 1, False)):
        torch.library.opcheck(ops.norm_bwd.default, args, test_utils=utils)


def test_one_device():
    x, w = rand(5, 32).cuda(), rand(32)
    ops = torch.ops.mamba_b200
    with pytest.raises(ValueError, match="one device"):
        ops.norm_fwd(x, None, None, w, None, 1e-5, 32, True, 0, False)
    with pytest.raises(ValueError, match="one device"):
        ops.norm_bwd(x, None, x, None, w, None, None, 1e-5, 32, True, 0, False)
