"""CUDA gated linear recurrence (scan, its gradients, the one-token step) against float64, step by step.

Tolerances: half a step of the output's type plus the float32 kernel's own error, counted in units
of 2^-24 of the largest value. A step of the recurrence rounds its decay (sigmoid, product with A,
exponential: at most 8 units at |A| <= 2), its input (two sigmoids, root, products: 16) and the sum
(1), and the joining of lanes and warps adds up to 10 products: 32 in all. Errors of earlier steps
decay with the state, so 1 + memory = 1 + 1 / (1 - mean decay) of them add up. A gradient goes
through both recurrences and up to six more factors: four times as much."""

import threading

import numpy as np
import pytest
import torch

import block_oracles as bo
import mamba_cpu_b200 as mb

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(b, d, L, dtype=F32, seed=0, initial=False, packed=False):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = dict(u=n(b, d, L).to(dtype), r=n(b, d, L).to(dtype), i=n(b, d, L).to(dtype),
             A=-0.1 - 1.9 * torch.rand(d, generator=g))
    x["h0"] = n(b, d) if initial else None
    x["ids"] = None
    if packed:
        ids = torch.cumsum(torch.rand(b, L, generator=g) < 0.05, 1)
        ids[torch.rand(b, L, generator=g) < 0.1] = -1
        if L > 3:
            ids[0, -L // 4:] = -1  # a padded tail
            ids[-1] = -1           # a row that is padding throughout
        x["ids"] = ids.to(torch.int32)
    x["dy"], x["dlast"] = n(b, d, L).to(dtype), n(b, d)
    return x


def want(x, grad=True):
    f = bo.f64
    return bo.scan(f(x["u"]), f(x["r"]), f(x["i"]), f(x["A"]), f(x["h0"]),
                   None if x["ids"] is None else x["ids"].numpy(), f(x["dy"]) if grad else None,
                   f(x["dlast"]) if grad else None)


NAMES = ("u", "r", "i", "A", "h0")


def cuda(x):
    return {k: None if v is None else v.cuda() for k, v in x.items()}


def run(x, grad=True):
    """(out, last) and the gradients by name, through the public function."""
    x = cuda(x)
    if not grad:
        return mb.gated_linear_scan_fn(x["u"], x["r"], x["i"], x["A"], x["h0"], x["ids"], True), None
    leaves = {k: x[k].detach().requires_grad_() for k in NAMES if x[k] is not None}
    out = mb.gated_linear_scan_fn(leaves["u"], leaves["r"], leaves["i"], leaves["A"], leaves.get("h0"), x["ids"], True)
    grads = torch.autograd.grad(out, list(leaves.values()), (x["dy"], x["dlast"]))
    return out, dict(zip(leaves, grads))


def compare(x, got, grads, ref, scale=1):
    dtype, L = x["u"].dtype, x["u"].shape[2]
    mem = 1 + bo.memory(ref, L)
    bo.check(got[0], ref["out"], dtype, scale * 32 * mem, name="out")
    bo.check(got[1], ref["last"], F32, scale * 32 * mem, name="last_state")
    if grads is None:
        return
    for n, k in (("u", "du"), ("r", "dr"), ("i", "di")):
        assert grads[n].dtype == dtype
        bo.check(grads[n], ref[k], dtype, scale * 128 * mem, name=k)
    bo.check(grads["A"], ref["dA"], F32, scale * 128 * mem, scale=ref["dA_abs"], name="dA")
    if x["h0"] is not None:
        bo.check(grads["h0"], ref["dh0"], F32, scale * 128 * mem, name="dh0")


@pytest.mark.parametrize("L", [1, 2, 7, 8, 9, 31, 255, 256, 257, 300, 512, 1000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_lengths(L, dtype):
    x = make(2, 5, L, dtype, seed=L, initial=L % 2 == 0)
    got, grads = run(x)
    compare(x, got, grads, want(x))


@pytest.mark.parametrize("b,d,L", [
    (1, 1, 1), (1, 1, 3000), (1, 3, 2049),   # one row over several warps and CTAs
    (1, 40, 5000), (2, 150, 600), (3, 700, 520),  # rows over 4 and 2 warps
    (2, 2500, 260),                          # a warp each
    (5, 13, 64),
])
@pytest.mark.parametrize("packed", [False, True])
def test_splits(b, d, L, packed):
    x = make(b, d, L, BF16 if d % 2 else F32, seed=d, initial=True, packed=packed)
    got, grads = run(x)
    compare(x, got, grads, want(x))


@pytest.mark.parametrize("b,d,L", [(1, 900, 1030), (2, 100, 4200), (1, 2, 9000), (1, 33, 4093), (3, 20, 4100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_splits_over_clusters(b, d, L, dtype):
    """Rows over 2, 8, 32 and 16 warps, packed and not."""
    for packed in (False, True):
        x = make(b, d, L, dtype, seed=d, initial=True, packed=packed)
        got, grads = run(x)
        compare(x, got, grads, want(x))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_inference_is_the_training_forward(dtype):
    x = make(2, 37, 777, dtype, initial=True, packed=True)
    (a, la), _ = run(x, grad=False)
    (b, lb), _ = run(x)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_packed_row_is_its_sequences():
    """A packed row gives the bits of its sequences run alone where they fall on the same lanes, and their
    values elsewhere."""
    x = make(1, 9, 600, F32, seed=3)
    ids = torch.zeros(1, 600, dtype=torch.int64)
    ids[:, 200:456], ids[:, 456:] = 7, 8
    xc = cuda(x)
    args = xc["u"], xc["r"], xc["i"]
    whole, last = mb.gated_linear_scan_fn(*args, xc["A"], seq_idx=ids.cuda(), return_last_state=True)
    parts = [mb.gated_linear_scan_fn(*[t[..., s:e] for t in args], xc["A"], return_last_state=True)
             for s, e in ((0, 200), (200, 456), (456, 600))]
    assert torch.equal(whole[..., :200], parts[0][0])
    torch.testing.assert_close(whole, torch.cat([p[0] for p in parts], -1), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(last, parts[2][1], rtol=1e-5, atol=1e-5)


def test_padding_hides_anything():
    """NaN, infinities and the type's lowest value in padded steps change nothing, in any direction."""
    x = make(3, 6, 530, F32, seed=5, initial=True, packed=True)
    ref, refg = run(x)
    pad = (x["ids"] < 0)[:, None].expand_as(x["u"])
    for bad in (float("nan"), float("inf"), torch.finfo(F32).min):
        y = {k: (torch.where(pad, torch.tensor(bad), v) if k in ("u", "r", "i", "dy") else v) for k, v in x.items()}
        got, grads = run(y)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        assert all(torch.equal(grads[k], refg[k]) for k in grads)
        assert not got[0][pad.cuda()].any() and not grads["r"][pad.cuda()].any()


def test_a_sequence_keeps_its_infinities():
    """NaN or infinity in one sequence of a row reaches neither its neighbours' outputs nor their gradients."""
    x = make(1, 4, 700, F32, seed=6)
    ids = torch.zeros(1, 700, dtype=torch.int32)
    ids[:, 300:450], ids[:, 450:] = 1, 2
    x["ids"] = ids
    ref, refg = run(x)
    keep = [slice(0, 300), slice(450, 700)]
    for bad in (float("nan"), float("inf")):
        y = dict(x, u=x["u"].clone(), dy=x["dy"].clone())
        y["u"][..., 320] = bad
        y["dy"][..., 400] = bad
        got, grads = run(y)
        assert not torch.isfinite(got[0][..., 320:450]).any()
        for s in keep:
            assert torch.equal(got[0][..., s], ref[0][..., s])
            assert all(torch.equal(grads[k][..., s], refg[k][..., s]) for k in ("u", "r", "i"))
        assert torch.equal(got[1], ref[1])


@pytest.mark.parametrize("b,d,L", [(1, 3, 1000), (3, 1000, 300)])  # rows over several warps, and a warp each
@pytest.mark.parametrize("A", [-3.0, -40.0, -400.0])
def test_a_sequence_does_not_lose_its_nan(b, d, L, A):
    """What is not a number stays so to the end of its sequence, and its gradient to the beginning, however fast the
    channel forgets: a product of decays that underflows, or a decay that does, is no start of a sequence."""
    x = make(b, d, L, F32, seed=8)
    x["A"] = torch.full((d,), A)
    x["u"][:, 1, 20] = float("nan")
    x["dy"][:, 2, L - 20] = float("nan")
    ids = torch.zeros(b, L, dtype=torch.int32)
    ids[:, 100:120], ids[:, L - 100:] = 1, 2  # marks in the first and the last chunk
    x["ids"] = ids
    got, grads = run(x)
    nan = torch.isnan(got[0]).cpu()
    want_nan = torch.zeros(b, d, L, dtype=torch.bool)
    want_nan[:, 1, 20:100] = True
    assert torch.equal(nan, want_nan)
    du = torch.zeros(b, d, L, dtype=torch.bool)
    du[:, 2, L - 100:L - 19] = True
    assert torch.equal(torch.isnan(grads["u"]).cpu(), du)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_extreme_gates(dtype):
    """Closed and open gates (infinite and at the type's limits), A of 0 and of -200."""
    x = make(1, 6, 40, dtype, seed=7, initial=True)
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    vals = torch.tensor([float("-inf"), float("inf"), lo, hi, -60.0, 60.0, -20.0, 20.0]).to(dtype)
    for k, name in enumerate(("r", "i")):
        for j in range(40):
            x[name][0, 1 + k:5, j] = vals[(j * (k + 1) + j // 8) % 8]
    x["A"][4:] = torch.tensor([0.0, -200.0])
    got, grads = run(x)
    # a channel whose gates stay shut never forgets: 40 steps of errors; |A| = 200 makes 100 times the error of |A| = 2
    # in a decay's exponent
    ref = want(x)
    compare(x, got, grads, ref, scale=100)
    # a channel with a shut decay gate everywhere keeps its state to the bit
    x["r"][0, 0] = float("-inf")
    got, _ = run(x, grad=False)
    assert torch.equal(got[0][0, 0].float(), x["h0"][0, :1].to(dtype).float().cuda().expand(40))
    assert torch.equal(got[1][0, 0], x["h0"][0, 0].cuda())


def test_long_memory():
    """Channels that forget next to nothing: |A| of 0.005 to 0.01 and decay gates around -8, 1 - a of 1e-6 to 6e-6.

    A step's decay is off by half a float32 step below 1, 2^-25: half a unit of 2^-24. Over a chunk of 256 steps a state
    takes 256 of those halves; its lane's 8 compositions, the 5 joins of the lanes and 5 of the warps round a partial sum
    (at most twice the largest state, as what two states differ by) and a product of decays: 18 (2 + 1), and 6 for the way
    in, 60. Inputs are off by 16 units each, decay gates by 12 of 1 - a. The recurrence of the gradients is the same from
    the other end; du's factors take 30 more."""
    d, L = 6, 4000
    x = make(1, d, L, seed=21, initial=True)
    x["A"] = -torch.linspace(0.005, 0.01, d)
    x["r"] = x["r"] * 0.25 - 8
    got, grads = run(x)
    ref = want(x)
    s_r, s_i = bo.sigmoid(bo.f64(x["r"])), bo.sigmoid(bo.f64(x["i"]))
    la = bo.f64(x["A"])[None, :, None] * s_r
    ms = np.sqrt(-np.expm1(2 * la)) * s_i
    assert 1e-7 < -la.max() and -la.min() < 1e-5
    own = 60 * (L // 256 + 2) + L / 2 + 12 * float(-la.sum(-1).min())
    top = max(np.abs(ref["out"]).max(), np.abs(bo.f64(x["h0"])).max())
    units = own + 16 * np.abs(ms * bo.f64(x["u"])).sum(-1).max() / top
    bo.check(got[0], ref["out"], F32, units, scale=top, name="out")
    bo.check(got[1], ref["last"], F32, units, scale=top, name="last_state")
    big = max(np.abs(ref["du"] / ms).max(), np.abs(bo.f64(x["dlast"])).max())  # the largest gradient of a state
    bo.check(grads["h0"], ref["dh0"], F32, own, scale=big, name="dh0")
    bo.check(grads["u"], ref["du"], F32, own + 30, scale=big * ms.max(), name="du")


def test_positive_A_is_nan():
    x = make(1, 2, 9, F32)
    x["A"][1] = 0.5
    (out, _), _ = run(x, grad=False)
    assert torch.isfinite(out[0, 0]).all() and torch.isnan(out[0, 1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype):
    """Slices, transposed and broadcast inputs, odd base addresses: the results are the dense ones.

    The chunks of a row follow the alignment of u's rows, so sums may be joined in another order: each result is
    within half a step + 32 (1 + memory) units of the exact one, and two results within the sum of two such limits."""
    b, d, L = 3, 10, 264
    cpu = make(b, d, L, dtype, seed=9, initial=True)
    mem = 1 + bo.memory(want(cpu, grad=False), L)
    x = cuda(cpu)
    dense = mb.gated_linear_scan_fn(x["u"], x["r"], x["i"], x["A"], x["h0"])

    def within(t, before, after, lead=1):  # t inside a larger array, rows of another length
        big = torch.full((b, d + lead, before + L + after), float("nan"), dtype=t.dtype, device="cuda")
        big[:, lead:, before:before + L] = t
        return big[:, lead:, before:before + L]

    forms = [
        (within(x["u"], 8, 8), within(x["r"], 16, 0), x["i"]),
        (within(x["u"], 1, 2), x["r"], within(x["i"], 3, 3)),
        (x["u"].transpose(1, 2).contiguous().transpose(1, 2), x["r"], x["i"]),
        (x["u"], x["r"].transpose(0, 1).contiguous().transpose(0, 1), x["i"]),
    ]
    for u, r, i in forms:
        bo.check(mb.gated_linear_scan_fn(u, r, i, x["A"], x["h0"]), bo.f64(dense), dtype, 2 * 32 * mem, halves=2)
    # broadcast over the batch, over channels and over steps, with gradients of the shared values
    for shape in ((1, d, L), (b, 1, L), (b, d, 1), (1, 1, 1)):
        r = x["r"][:shape[0], :shape[1], :shape[2]].clone().requires_grad_()
        u = x["u"].clone().requires_grad_()
        y = mb.gated_linear_scan_fn(u, r.expand(b, d, L), x["i"], x["A"], x["h0"])
        gr, gu = torch.autograd.grad(y, (r, u), x["dy"])
        full = r.detach().expand(b, d, L).contiguous().requires_grad_()
        y2 = mb.gated_linear_scan_fn(u, full, x["i"], x["A"], x["h0"])
        g2, gu2 = torch.autograd.grad(y2, (full, u), x["dy"])
        assert torch.equal(y, y2) and torch.equal(gu, gu2) and gr.shape == r.shape
        dims = [k for k in range(3) if shape[k] == 1 and (b, d, L)[k] > 1]
        torch.testing.assert_close(gr, g2.sum(dims, keepdim=True), rtol=2e-2 if dtype == BF16 else 1e-4, atol=1e-3)


def test_mixed_and_other_types():
    x = cuda(make(2, 5, 70, F32, initial=True))
    y = mb.gated_linear_scan_fn(x["u"].to(BF16), x["r"], x["i"], x["A"].double(), x["h0"].to(BF16))
    w = mb.gated_linear_scan_fn(x["u"].to(BF16).float(), x["r"], x["i"], x["A"], x["h0"].to(BF16).float())
    assert y.dtype == BF16 and torch.equal(y, w.to(BF16))
    u = x["u"].double().requires_grad_()
    y = mb.gated_linear_scan_fn(u, x["r"].double(), x["i"].double(), x["A"])
    g, = torch.autograd.grad(y, u, x["dy"].double())
    assert y.dtype == torch.float64 and g.dtype == torch.float64


@pytest.mark.parametrize("shape", [(0, 4, 8), (2, 0, 8), (2, 4, 0), (0, 0, 0)])
def test_empty(shape):
    x = make(*shape, initial=True)
    (out, last), grads = run(x)
    assert out.shape == shape and last.shape == shape[:2]
    assert not grads["A"].any()
    if shape[2] == 0:
        assert torch.equal(last.cpu(), x["h0"]) and torch.equal(grads["h0"].cpu(), x["dlast"])


def test_partial_gradients():
    """Only some inputs ask for gradients; only one output has one."""
    x = cuda(make(2, 6, 300, F32, initial=True))
    A = x["A"].clone().requires_grad_()
    y, last = mb.gated_linear_scan_fn(x["u"], x["r"], x["i"], A, return_last_state=True)
    gA, = torch.autograd.grad(y, A, x["dy"], retain_graph=True)
    gL, = torch.autograd.grad(last, A, x["dlast"], retain_graph=True)
    both, = torch.autograd.grad((y, last), A, (x["dy"], x["dlast"]))
    torch.testing.assert_close(gA + gL, both, rtol=1e-4, atol=1e-4)


def test_gradient_against_differences():
    """The kernel's gradients along a direction against central differences of the float64 forward."""
    x = make(2, 7, 290, F32, seed=11, initial=True, packed=True)
    _, grads = run(x)
    rng = np.random.default_rng(0)
    vals = {k: bo.f64(x[k]) for k in NAMES}
    dy, dlast, ids = bo.f64(x["dy"]), bo.f64(x["dlast"]), x["ids"].numpy()

    def f(v):
        r = bo.scan(v["u"], v["r"], v["i"], v["A"], v["h0"], ids)
        return (r["out"] * dy).sum() + (r["last"] * dlast).sum()

    for k in NAMES:
        v, h = rng.standard_normal(vals[k].shape), 1e-6
        diff = (f({**vals, k: vals[k] + h * v}) - f({**vals, k: vals[k] - h * v})) / (2 * h)
        terms = bo.f64(grads[k]) * v
        # the gradients' own tolerance, on terms whose signs are random
        assert abs(diff - terms.sum()) <= 1e-5 * np.abs(terms).sum() + 1e-6, k


def test_steps_are_the_scan():
    x = cuda(make(3, 33, 40, F32, initial=True))
    out, last = mb.gated_linear_scan_fn(x["u"], x["r"], x["i"], x["A"], x["h0"], return_last_state=True)
    state = x["h0"].clone()
    ys = [mb.gated_linear_scan_update(state, x["u"][..., t], x["r"][..., t], x["i"][..., t], x["A"]) for t in range(40)]
    torch.testing.assert_close(torch.stack(ys, -1), out, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype,state_dtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16),
                                               (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("b,d", [(1, 1), (3, 130), (2, 1536), (65, 7)])
def test_step(dtype, state_dtype, b, d):
    x = make(b, d, 1, dtype, seed=d, initial=True)
    state = x["h0"].to(state_dtype)
    ref = bo.scan(*[bo.f64(x[k]) for k in ("u", "r", "i", "A")], bo.f64(state))["last"]
    xc = {k: x[k][..., 0].cuda() for k in ("u", "r", "i")}
    sg = state.cuda()
    y = mb.gated_linear_scan_update(sg, xc["u"], xc["r"], xc["i"], x["A"].cuda())
    bo.check(y, ref, dtype, 64, name="out")
    bo.check(sg, ref, state_dtype, 64, name="state")
    # out of place: the old state stays, the new one is the same
    s0, s1 = state.cuda(), torch.full_like(sg, float("nan"))
    y2 = mb.gated_linear_scan_update(s0, xc["u"], xc["r"], xc["i"], x["A"].cuda(), out_state=s1)
    assert torch.equal(s0.cpu(), state) and torch.equal(s1, sg) and torch.equal(y2, y)


def test_step_layouts():
    x = cuda(make(4, 24, 1, F32, initial=True))
    u, r, i, A, h0 = x["u"][..., 0], x["r"][..., 0], x["i"][..., 0], x["A"], x["h0"]
    state = h0.clone()
    y = mb.gated_linear_scan_update(state, u, r, i, A)
    cache = torch.full((4, 3, 24), float("nan"), device="cuda")
    cache[:, 1] = h0
    assert torch.equal(mb.gated_linear_scan_update(cache[:, 1], u, r, i, A), y)
    assert torch.equal(cache[:, 1], state) and torch.isnan(cache[:, [0, 2]]).all()
    cache[:, 1] = h0
    assert torch.equal(mb.gated_linear_scan_update(cache[:, 1], u, r, i, A, out_state=cache[:, 2]), y)
    assert torch.equal(cache[:, 1], h0) and torch.equal(cache[:, 2], state) and torch.isnan(cache[:, 0]).all()
    t = h0.t().contiguous().t()  # columns contiguous
    assert torch.equal(mb.gated_linear_scan_update(t, u.t().contiguous().t(), r, i, A), y) and torch.equal(t, state)
    odd = torch.full((4, 27), float("nan"), device="cuda")
    odd[:, 1:25] = h0
    assert torch.equal(mb.gated_linear_scan_update(odd[:, 1:25], u, r, i, A), y) and torch.equal(odd[:, 1:25], state)
    assert torch.isnan(odd[:, [0, 25, 26]]).all()
    new = torch.empty_like(h0)
    zero = mb.gated_linear_scan_update(torch.zeros(1, 24, device="cuda").expand(4, 24), u, r, i, A, out_state=new)
    assert torch.equal(zero, new)
    assert torch.equal(mb.gated_linear_scan_update(h0, u[:1].expand(4, 24), r, i, A, out_state=new)[:1], y[:1])
    buf = torch.zeros(5, 24, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        mb.gated_linear_scan_update(buf[:4], u, r, i, A, out_state=buf[1:])
    with pytest.raises(ValueError, match="overlap"):
        mb.gated_linear_scan_update(h0, buf[:4], r, i, A, out_state=buf[1:])
    with pytest.raises(ValueError, match="overlap"):
        mb.gated_linear_scan_update(buf[:4], u, r, i, buf[2])
    packed = torch.cat([h0, u, r, i], 1)  # state and inputs side by side in one buffer
    assert torch.equal(mb.gated_linear_scan_update(*packed.chunk(4, 1), A), y) and torch.equal(packed[:, :24], state)
    empty = torch.zeros(0, 24, device="cuda")
    assert mb.gated_linear_scan_update(empty, empty, empty, empty, A).shape == (0, 24)


def _step_call(x):
    leaves = [x[k].detach().requires_grad_() for k in NAMES]

    def call():
        y, last = mb.gated_linear_scan_fn(*leaves[:4], leaves[4], x["ids"], True)
        return (y, last) + torch.autograd.grad((y, last), leaves, (x["dy"], x["dlast"]))

    return call


def test_captured_and_replayed():
    """Two graphs captured side by side, forward and backward, replayed in turn on changed inputs."""
    xs = [cuda(make(2, 70, 900, BF16, seed=s, initial=True, packed=s == 1)) for s in range(2)]
    calls = [_step_call(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c())
        graphs.append(g)
    for turn in range(2):
        for x in xs:
            x["u"].mul_(-0.5)
            x["dy"].add_(0.25)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c, o in zip(calls, outs):
            assert all(torch.equal(a, b) for a, b in zip(c(), o))


def test_streams_and_threads():
    """Calls on several streams from several threads at once give the bits of calls in turn."""
    calls = [_step_call(cuda(make(2, 50, 1300, F32, seed=s, initial=True))) for s in range(4)]
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


def test_first_order_only():
    """Gradients that are asked to be differentiable come, and raise when they are differentiated."""
    x = cuda(make(1, 3, 20, F32))
    leaf = x["u"].clone().requires_grad_()
    g, = torch.autograd.grad(mb.gated_linear_scan_fn(leaf, x["r"], x["i"], x["A"]), leaf, x["dy"], create_graph=True)
    ref, = torch.autograd.grad(mb.gated_linear_scan_fn(leaf, x["r"], x["i"], x["A"]), leaf, x["dy"])
    assert torch.equal(g, ref)
    if g.requires_grad:
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaf)


def test_second_backward_raises():
    """A gradient that was asked to be differentiable says so, and differentiating it raises, whichever input it is of."""
    x = cuda(make(2, 3, 20, F32, initial=True))
    leaves = [x[k].requires_grad_() for k in NAMES]
    y = mb.gated_linear_scan_fn(*leaves)
    for g in torch.autograd.grad(y, leaves, x["dy"], create_graph=True):
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="gated_scan_bwd is not implemented"):
            torch.autograd.grad(g.sum(), leaves[0], retain_graph=True)


def test_compiled():
    """Traced and run by torch.compile's eager backend: forward, gradients and the step."""
    x = cuda(make(2, 6, 300, F32, initial=True, packed=True))

    def f(u, r, i, A, h0):
        y, last = mb.gated_linear_scan_fn(u, r, i, A, h0, x["ids"], True)
        return y * 2, last

    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    want_ = f(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want_))
    ga, gb = (torch.autograd.grad(o, leaves, (x["dy"], x["dlast"])) for o in (got, want_))
    assert all(torch.equal(a, b) for a, b in zip(ga, gb))
    s1, s2 = x["h0"].clone(), x["h0"].clone()
    step = lambda s: mb.gated_linear_scan_update(s, x["u"][..., 0], x["r"][..., 0], x["i"][..., 0], x["A"])  # noqa: E731
    assert torch.equal(torch.compile(step, backend="aot_eager")(s1), step(s2)) and torch.equal(s1, s2)


@pytest.mark.slow
def test_offsets_past_32_bits():
    """More than 2^31 elements a tensor: the last rows are those of a call on them alone."""
    b, d, L = 1, 36000, 60000
    g = torch.Generator(device="cuda").manual_seed(0)
    u, r, i, dy = (torch.empty(b, d, L, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(4))
    A = -torch.rand(d, generator=g, device="cuda")
    leaves = [t.requires_grad_() for t in (u, r, i, A)]
    y = mb.gated_linear_scan_fn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    tail = [t.detach()[:, -3:].contiguous().requires_grad_() for t in leaves[:3]] + [A.detach()[-3:].clone().requires_grad_()]
    y2 = mb.gated_linear_scan_fn(*tail)
    g2 = torch.autograd.grad(y2, tail, dy[:, -3:].contiguous())
    # the tail's rows may be shared by more warps, which join them in another order
    torch.testing.assert_close(y[:, -3:], y2, rtol=2e-2, atol=1e-3)
    for a, c in zip(grads[:3], g2):
        torch.testing.assert_close(a[:, -3:], c, rtol=2e-2, atol=2e-3)
    torch.testing.assert_close(grads[3][-3:], g2[3], rtol=1e-3, atol=1e-2)


@pytest.mark.parametrize("per_sm", [31, 35, 44, 47])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_rows_in_waves(dtype, per_sm):
    """Long rows, a warp each: the bits do not depend on how many run at a time, with ids or without."""
    d, L = 148 * per_sm - 5, 8200
    g = torch.Generator(device="cuda").manual_seed(per_sm)
    u, r, i = (torch.randn(1, d, L, device="cuda", generator=g).to(dtype) for _ in range(3))
    A = -torch.rand(d, generator=g, device="cuda")
    ids = (torch.arange(L, device="cuda") // 1000)[None].to(torch.int32)
    for seq in (None, ids):
        whole = mb.gated_linear_scan_fn(u, r, i, A, seq_idx=seq)
        for s in (slice(0, d // 2), slice(d // 2, d)):
            # (each half is more rows than 14 an SM, so a warp each too)
            assert torch.equal(whole[:, s], mb.gated_linear_scan_fn(u[:, s], r[:, s], i[:, s], A[s], seq_idx=seq))


def test_opcheck():
    x = cuda(make(2, 5, 300, BF16, initial=True, packed=True))
    ops, utils = torch.ops.mamba_b200, ("test_schema", "test_faketensor")
    args = (x["u"], x["r"], x["i"], x["A"], x["h0"], x["ids"])
    for save in (False, True):
        torch.library.opcheck(ops.gated_scan_fwd.default, args + (save,), test_utils=utils)
    states = ops.gated_scan_fwd(*args, True)[2]
    torch.library.opcheck(ops.gated_scan_bwd.default, args + (states, x["dy"], x["dlast"]), test_utils=utils)
    step = tuple(x[k][..., 0].contiguous() for k in ("u", "r", "i")) + (x["A"],)
    torch.library.opcheck(ops.gated_scan_update.default, (x["h0"].clone(),) + step, test_utils=utils)
    torch.library.opcheck(ops.gated_scan_update_out.default, (x["h0"],) + step + (torch.empty_like(x["h0"]),),
                          test_utils=utils)


def test_one_device():
    x = cuda(make(2, 5, 30, F32, initial=True))
    ops, args = torch.ops.mamba_b200, (x["u"], x["r"], x["i"])
    with pytest.raises(ValueError, match="one device"):
        ops.gated_scan_fwd(*args, x["A"].cpu(), x["h0"], None, True)
    with pytest.raises(ValueError, match="one device"):
        ops.gated_scan_update(x["h0"], *(t[..., 0] for t in args), x["A"].cpu())
