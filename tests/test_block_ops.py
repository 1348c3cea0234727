"""The gated linear recurrence and the norms without a GPU: C ABI argument checks and struct layouts,
refusals and shapes of the public functions on fake CUDA tensors, and the oracles' gradients against
differences."""

import ctypes
import os
import shutil
import subprocess
import sys
import tempfile

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import block_oracles as bo
import mamba_cpu_b200 as mb
from mamba_cpu_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_STRUCTS = {
    "mb200_gated_scan_params": _lib.GatedScanParams,
    "mb200_gated_scan_bwd_params": _lib.GatedScanBwdParams,
    "mb200_gated_step_params": _lib.GatedStepParams,
    "mb200_norm_params": _lib.NormParams,
    "mb200_norm_bwd_params": _lib.NormBwdParams,
}


def test_struct_layout_and_constants_match_header():
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mamba_b200.h"', "int main(void) {"]
    for cname, py in _STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'printf("{cname}.{fname} %zu\\n", offsetof({cname}, {fname}));')
    consts = dict(MB200_GATED_SCAN_CHUNK=_lib.GATED_SCAN_CHUNK, MB200_NORM_MAX_DIM=_lib.NORM_MAX_DIM,
                  MB200_GATE_NONE=_lib.GATE_NONE, MB200_GATE_AFTER_NORM=_lib.GATE_AFTER_NORM,
                  MB200_GATE_BEFORE_NORM=_lib.GATE_BEFORE_NORM)
    lines += [f'printf("{c} %d\\n", {c});' for c in consts] + ["return 0; }"]
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "probe.c"), os.path.join(td, "probe")
        with open(src, "w") as f:
            f.write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = dict(l.split() for l in subprocess.run([exe], capture_output=True, text=True, check=True)
                   .stdout.splitlines())
    for cname, py in _STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(py), cname
        for fname, _ in py._fields_:
            assert int(got[f"{cname}.{fname}"]) == getattr(py, fname).offset, f"{cname}.{fname}"
    for c, v in consts.items():
        assert int(got[c]) == v, c


# ---- C ABI: every refusal comes before any CUDA work, so these need no GPU --------------------------


def _set(p, kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _scan_params(**kw):
    p = _lib.GatedScanParams()
    p.u = p.decay_gate = p.input_gate = p.A = p.out = 0x1000
    p.batch, p.dim, p.seqlen = 2, 4, 8
    return _set(p, kw)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 2), (dict(dim=-1), 2), (dict(seqlen=-1), 2), (dict(io_dtype=3), 3), (dict(u=None), 1),
    (dict(decay_gate=None), 1), (dict(input_gate=None), 1), (dict(A=None), 1), (dict(out=None), 1),
    (dict(u_batch_stride=-8), 4), (dict(input_gate_dim_stride=-8), 4), (dict(seq_idx_batch_stride=-1), 4),
    (dict(batch=1 << 20, dim=1 << 20), 5), (dict(seqlen=1 << 45), 5),
    (dict(batch=1 << 62, dim=4), 5), (dict(batch=1 << 32, dim=1 << 32), 5),
])
def test_scan_refusals(kw, status):
    assert _lib.lib.mb200_gated_scan_fwd(_scan_params(**kw), None) == status


def test_scan_bwd_refusals():
    p = _lib.GatedScanBwdParams()
    p.fwd = _scan_params(chunk_states=0x1000)
    p.dout = p.du = p.ddecay_gate = p.dinput_gate = p.dA = 0x1000
    need = _lib.lib.mb200_gated_scan_bwd_workspace_size(p)
    assert need == 256  # 2 x 4 floats
    assert _lib.lib.mb200_gated_scan_bwd(p, None, 0, None) == 6
    assert _lib.lib.mb200_gated_scan_bwd(p, 0x1000, need - 1, None) == 6
    assert _lib.lib.mb200_gated_scan_bwd(p, 0x1010, need, None) == 6
    for name in ("dout", "du", "ddecay_gate", "dinput_gate", "dA"):
        setattr(p, name, None)
        assert _lib.lib.mb200_gated_scan_bwd(p, 0x1000, need, None) == 1, name
        assert _lib.lib.mb200_gated_scan_bwd_workspace_size(p) == 0
        setattr(p, name, 0x1000)
    p.fwd.chunk_states = None
    assert _lib.lib.mb200_gated_scan_bwd(p, 0x1000, need, None) == 1
    p.fwd = _scan_params(chunk_states=0x1000, batch=1)
    assert _lib.lib.mb200_gated_scan_bwd_workspace_size(p) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 2), (dict(io_dtype=5), 3), (dict(io_dtype=1, state_dtype=2), 3), (dict(state=None), 1),
    (dict(new_state=None), 1), (dict(u=None), 1), (dict(A=None), 1), (dict(out=None), 1), (dict(u_stride=-1), 4),
    (dict(state_stride=3), 4), (dict(new_state_stride=3), 4), (dict(state_stride=8), 4),
    (dict(batch=1 << 28, dim=1 << 20), 5),
])
def test_step_refusals(kw, status):
    p = _lib.GatedStepParams()
    p.state = p.new_state = p.u = p.decay_gate = p.input_gate = p.A = p.out = 0x1000
    p.batch, p.dim = 2, 4
    assert _lib.lib.mb200_gated_scan_update(_set(p, kw), None) == status


def _norm_params(**kw):
    p = _lib.NormParams()
    p.x = p.weight = p.out = 0x1000
    p.rows, p.dim, p.group_size, p.eps = 2, 8, 8, 1e-5
    return _set(p, kw)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), 2), (dict(dim=-1), 2), (dict(group_size=0), 2), (dict(group_size=4), 2), (dict(gate=3), 2),
    (dict(gate=-1), 2), (dict(eps=-1.0), 2), (dict(eps=float("nan")), 2), (dict(io_dtype=3), 3),
    (dict(weight_dtype=1), 3), (dict(residual=0x1000, residual_dtype=2), 3), (dict(x=None), 1), (dict(out=None), 1),
    (dict(gate=1, rms=1, group_size=4), 1), (dict(gate=1, rms=0, z=0x1000), 5),
    (dict(gate=2, rms=1, z=0x1000, bias=0x1000), 5), (dict(gate=2, rms=1, z=0x1000, residual=0x1000), 5),
    (dict(gate=2, rms=1, z=0x1000, group_size=3), 2), (dict(dim=16385, group_size=16385), 5),
    (dict(gate=1, rms=1, z=0x1000, dim=65536, group_size=1), 5), (dict(x_stride=-8), 4),
    (dict(residual=0x1000, residual_stride=-8), 4),
])
def test_norm_refusals(kw, status):
    assert _lib.lib.mb200_norm_fwd(_norm_params(**kw), None) == status


def test_norm_bwd_refusals():
    p = _lib.NormBwdParams()
    p.fwd = _norm_params()
    p.dout = p.dx = p.dweight = 0x1000
    assert _lib.lib.mb200_norm_bwd_workspace_size(p) == 0  # two rows are one CTA's, which needs none
    p.fwd = _norm_params(rows=1 << 20)
    need = _lib.lib.mb200_norm_bwd_workspace_size(p)
    assert need >= 2 * 8 * 4 and need % 256 == 0
    assert _lib.lib.mb200_norm_bwd(p, None, 0, None) == 6
    assert _lib.lib.mb200_norm_bwd(p, 0x1000, need - 1, None) == 6
    assert _lib.lib.mb200_norm_bwd(p, 0x1008, need, None) == 6
    p.dx = None
    assert _lib.lib.mb200_norm_bwd(p, 0x1000, need, None) == 1
    p.dx, p.fwd = 0x1000, _norm_params(gate=1, rms=1, z=0x1000, group_size=4)
    assert _lib.lib.mb200_norm_bwd(p, 0x1000, need, None) == 1  # dz missing
    p.fwd, p.dweight = _norm_params(rows=1 << 20), None
    assert _lib.lib.mb200_norm_bwd_workspace_size(p) == 0


@pytest.mark.parametrize("dim", [5, 64, 256, 511, 512, 2048, 5120, 16383])
def test_norm_workspace_of_any_alignment(dim):
    """The size that is asked for with one set of addresses is enough for others."""
    p = _lib.NormBwdParams()
    p.fwd = _norm_params(rows=1000, dim=dim, group_size=dim, rms=1, io_dtype=1)
    p.dout = p.dx = p.dweight = 0x1000
    size = _lib.lib.mb200_norm_bwd_workspace_size(p)
    assert size > 0
    for off in (2, 8, 14):
        p.dx = 0x1000 + off
        assert _lib.lib.mb200_norm_bwd_workspace_size(p) == size
        p.fwd.x = 0x1000 + off
        assert _lib.lib.mb200_norm_bwd_workspace_size(p) == size
        p.dx, p.fwd.x = 0x1000, 0x1000


def test_library_from_another_place():
    """MAMBA_B200_LIB names a library that lies alone: the package's torch binding loads, and calls that library."""
    with tempfile.TemporaryDirectory() as td:
        other = os.path.join(td, "libmamba_b200.so")
        shutil.copy(os.path.join(os.path.dirname(_lib.__file__), "_lib", "libmamba_b200.so"), other)
        code = ("import mamba_cpu_b200 as mb, torch; from mamba_cpu_b200 import _lib; torch.ops.mamba_b200.norm.default;"
                "print(_lib.lib._name); print(*sorted({l.split()[-1] for l in open('/proc/self/maps')"
                " if 'libmamba_b200.so' in l}))")
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                           env=dict(os.environ, MAMBA_B200_LIB=other, PYTHONPATH=os.path.join(ROOT, "mamba-cpu_b200")))
        assert r.returncode == 0, r.stderr
        assert r.stdout.split() == [other, other]


# ---- the public functions on fake CUDA tensors ---------------------------------------------------------


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4)
    for call in (lambda: mb.gated_linear_scan_fn(x[None], x[None], x[None], x[0]),
                 lambda: mb.gated_linear_scan_update(x, x, x, x, x[0]), lambda: mb.layer_norm_fn(x, x[0]),
                 lambda: mb.rms_norm_fn(x, x[0]), lambda: mb.gated_rms_norm_fn(x, x, x[0])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _fake(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


_REFUSED = [
    (lambda x: mb.gated_linear_scan_fn(_fake(2, 4), _fake(2, 4), _fake(2, 4), _fake(4)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, _fake(2, 4, 7), x, _fake(4)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, x, _fake(1, 4, 8), _fake(4)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4, 1)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4, dtype=torch.complex64)), NotImplementedError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4), _fake(2, 4, 1)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4), seq_idx=_fake(2, 7, dtype=torch.int32)), ValueError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4), seq_idx=_fake(2, 8)), TypeError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, _fake(4), seq_idx=_fake(2, 8, dtype=torch.bool)), TypeError),
    (lambda x: mb.gated_linear_scan_fn(x, x, x, torch.empty(4, device="meta")), ValueError),
    (lambda x: mb.gated_linear_scan_update(x[0], x[0], x[0], x[0], _fake(4)), ValueError),
    (lambda x: mb.gated_linear_scan_update(_fake(4, 7), x[0], x[0], x[0], _fake(8)), ValueError),
    (lambda x: mb.gated_linear_scan_update(x, x, x, x, _fake(8)), ValueError),
    (lambda x: mb.gated_linear_scan_update(_fake(1, 8).expand(4, 8), x[0], x[0], x[0], _fake(8)), ValueError),
    (lambda x: mb.gated_linear_scan_update(_fake(4, 1).expand(4, 8), x[0], x[0], x[0], _fake(8)), ValueError),
    (lambda x: mb.gated_linear_scan_update(_fake(32).as_strided((4, 8), (4, 1)), x[0], x[0], x[0], _fake(8)),
     ValueError),
    (lambda x: mb.gated_linear_scan_update(x[0], x[0], x[0], x[0], _fake(8),
                                           out_state=_fake(4, 8, dtype=torch.bfloat16)), TypeError),
    (lambda x: mb.layer_norm_fn(x, _fake(7)), ValueError),
    (lambda x: mb.layer_norm_fn(x, _fake(8), _fake(4)), ValueError),
    (lambda x: mb.rms_norm_fn(x, _fake(8), residual=_fake(2, 8)), ValueError),
    (lambda x: mb.rms_norm_fn(x, _fake(8), eps=-1e-5), ValueError),
    (lambda x: mb.rms_norm_fn(x, _fake(8), eps=float("nan")), ValueError),
    (lambda x: mb.rms_norm_fn(_fake(()), None), ValueError),
    (lambda x: mb.rms_norm_fn(_fake(2, 16385), None), NotImplementedError),
    (lambda x: mb.rms_norm_fn(x, torch.empty(8, device="meta")), ValueError),
    (lambda x: mb.gated_rms_norm_fn(x, _fake(2, 4, 4), _fake(8)), ValueError),
    (lambda x: mb.gated_rms_norm_fn(x, x, _fake(8), group_size=3), ValueError),
    (lambda x: mb.gated_rms_norm_fn(x, x, _fake(8), group_size=0), ValueError),
    (lambda x: mb.gated_rms_norm_fn(x, x, _fake(8), group_size=-8), ValueError),
    (lambda x: mb.gated_rms_norm_fn(_fake(2, 65536), _fake(2, 65536), None, group_size=1), NotImplementedError),
    (lambda x: mb.gated_rms_norm_fn(_fake(2, 32768), _fake(2, 32768), None), NotImplementedError),
]


@pytest.mark.parametrize("i", range(len(_REFUSED)))
def test_refusals(i):
    call, exc = _REFUSED[i]
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(exc):
            call(_fake(2, 4, 8))


def test_shapes_and_dtypes_on_fake_tensors():
    bf = torch.bfloat16
    with FakeTensorMode():
        u, A = _fake(2, 4, 300, dtype=bf), _fake(4)
        y, last = mb.gated_linear_scan_fn(u, u, u, A, return_last_state=True)
        assert y.shape == u.shape and y.dtype == bf and last.shape == (2, 4) and last.dtype == torch.float32
        leaf = _fake(2, 4, 300, dtype=bf).requires_grad_()
        y = mb.gated_linear_scan_fn(leaf, u, u, A.requires_grad_(), _fake(2, 4))
        assert y.grad_fn is not None
        ops = torch.ops.mamba_b200
        got = ops.gated_scan_bwd(u, u, u, _fake(4), _fake(2, 4), None, _fake(20), u, None)
        assert [t.shape for t in got] == [u.shape] * 3 + [(4,), (2, 4)] and got[0].dtype == bf
        st = _fake(2, 4, dtype=bf)
        assert mb.gated_linear_scan_update(st, u[..., 0], u[..., 0], u[..., 0], A).dtype == bf
        x, r, w = _fake(3, 5, 16, dtype=bf).requires_grad_(), _fake(3, 5, 16), _fake(16).requires_grad_()
        y, s = mb.rms_norm_fn(x, w, residual=r, prenorm=True)
        assert y.dtype == bf and s.dtype == torch.float32 and s.shape == x.shape
        assert y.grad_fn is not None and s.grad_fn is not None
        got = ops.norm_bwd(y.detach(), s.detach(), s.detach(), None, w.detach(), torch.float32, torch.float32, 1e-5, 16,
                           True, 0, True)
        assert [(t.shape, t.dtype) for t in got] == [(x.shape, bf), (x.shape, torch.float32), ((0,), bf),
                                                     ((16,), torch.float32), ((16,), torch.float32)]
        y, s = mb.layer_norm_fn(x, w, residual=r.to(bf), prenorm=True)
        assert s.dtype == bf
        y, s = mb.layer_norm_fn(x, w, prenorm=True, residual_in_fp32=True)
        assert s.dtype == torch.float32
        y = mb.gated_rms_norm_fn(x, x.detach(), w, group_size=4)
        assert y.grad_fn is not None and y.shape == x.shape
        got = ops.norm_bwd(y.detach(), None, x.detach(), x.detach(), w.detach(), None, None, 1e-5, 4, True, 1, False)
        assert [t.shape for t in got] == [x.shape, (0,), x.shape, (16,), (0,)]


_TENSORS = {  # every tensor argument by name, and the call
    "scan": (dict(u=(2, 4, 8), r=(2, 4, 8), i=(2, 4, 8), A=(4,), h0=(2, 4)),
             lambda t: mb.gated_linear_scan_fn(t["u"], t["r"], t["i"], t["A"], t["h0"])),
    "step": (dict(state=(2, 4), u=(2, 4), r=(2, 4), i=(2, 4), A=(4,)),
             lambda t: mb.gated_linear_scan_update(t["state"], t["u"], t["r"], t["i"], t["A"])),
    "step to": (dict(state=(2, 4), u=(2, 4), out_state=(2, 4), A=(4,)),
                lambda t: mb.gated_linear_scan_update(t["state"], t["u"], t["u"], t["u"], t["A"], t["out_state"])),
    "layer norm": (dict(x=(3, 8), w=(8,), b=(8,), res=(3, 8)),
                   lambda t: mb.layer_norm_fn(t["x"], t["w"], t["b"], t["res"])),
    "rms norm": (dict(x=(3, 8), w=(8,), b=(8,), res=(3, 8)),
                 lambda t: mb.rms_norm_fn(t["x"], t["w"], t["b"], t["res"], prenorm=True)[1]),
    "gated norm": (dict(x=(3, 8), z=(3, 8), w=(8,)), lambda t: mb.gated_rms_norm_fn(t["x"], t["z"], t["w"])),
}


@pytest.mark.parametrize("name,arg", [(n, a) for n, (shapes, _) in _TENSORS.items() for a in shapes])
def test_complex_tensors_are_refused(name, arg):
    """No argument loses its imaginary part on the way to float32."""
    shapes, call = _TENSORS[name]
    with FakeTensorMode():
        t = {k: _fake(*s) for k, s in shapes.items()}
        t[arg] = _fake(*shapes[arg], dtype=torch.complex64)
        if arg == "state" and "out_state" in t:
            t["out_state"] = _fake(*shapes["out_state"], dtype=torch.complex64)
        with pytest.raises((TypeError, NotImplementedError)):
            call(t)


@pytest.mark.parametrize("name,arg", [("scan", "u"), ("step", "u"), ("step", "state"), ("layer norm", "x"),
                                      ("rms norm", "x"), ("gated norm", "x")])
@pytest.mark.parametrize("dtype", [torch.int32, torch.bool])
def test_results_are_not_cut_to_integers(name, arg, dtype):
    """The argument whose type a result takes is of floating point."""
    shapes, call = _TENSORS[name]
    with FakeTensorMode():
        t = {k: _fake(*s) for k, s in shapes.items()}
        with pytest.raises(TypeError, match="floating point"):
            call({**t, arg: _fake(*shapes[arg], dtype=dtype)})


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("b,l", [(1, 12), (3, 12)])
def test_mixer_delta_is_read_in_place(monkeypatch, rms, b, l):
    """mamba_inner_fn hands the scan a delta whose (b, d, l) view has contiguous rows, with delta's norm and without."""
    from mamba_cpu_b200 import hf

    d, n, r, dm, seen = 32, 4, 2, 16, []

    def scan(u, delta, *rest):
        seen.append(delta)
        return u

    monkeypatch.setattr(hf, "causal_conv1d_fn", lambda x, w, bias, activation: x.contiguous())
    monkeypatch.setattr(hf, "selective_scan_fn", scan)
    bf = torch.bfloat16
    with FakeTensorMode():
        y = hf.mamba_inner_fn(_fake(b, 2 * d, l, dtype=bf), _fake(d, 1, 4, dtype=bf), None, _fake(r + 2 * n, d, dtype=bf),
                              _fake(d, r, dtype=bf), _fake(dm, d, dtype=bf), None, _fake(d, n),
                              dt_rms_weight=_fake(d, dtype=bf) if rms else None)
    delta, = seen
    assert y.shape == (b, l, dm) and delta.shape == (b, d, l) and delta.dtype == bf
    assert delta.stride()[1:] == (b * l, 1) and (b == 1 or delta.stride(0) == l)


@pytest.mark.parametrize("name,arg", [(n, a) for n, (shapes, _) in _TENSORS.items() for a in shapes])
def test_forward_mode_is_refused(name, arg):
    """A tangent on any argument raises, with gradients enabled or not: none comes back as zero."""
    shapes, call = _TENSORS[name]
    with FakeTensorMode():
        t = {k: _fake(*s) for k, s in shapes.items()}
        direction = _fake(*shapes[arg])
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                with fwAD.dual_level():
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call({**t, arg: fwAD.make_dual(t[arg], direction)})
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.func.jvp(lambda v: call({**t, arg: v}), (t[arg],), (direction,))
        with fwAD.dual_level():  # no argument has one
            call(t)


# ---- the oracles' gradients against differences ---------------------------------------------------------


def _difference(f, args, grads, rng, h=1e-6):
    """Central difference of f along a random direction against the gradients' products with it."""
    dirs = [rng.standard_normal(a.shape) for a in args]
    plus = f(*[a + h * v for a, v in zip(args, dirs)])
    minus = f(*[a - h * v for a, v in zip(args, dirs)])
    want = (plus - minus) / (2 * h)
    got = sum((g * v).sum() for g, v in zip(grads, dirs))
    # truncation h^2 and cancellation 2^-53 / h, both below 1e-8 of the terms' size
    assert abs(got - want) <= 1e-6 * max(1.0, sum(np.abs(g * v).sum() for g, v in zip(grads, dirs)))


@pytest.mark.parametrize("packed", [False, True])
def test_scan_oracle_gradient(packed):
    rng = np.random.default_rng(0)
    b, d, L = 2, 3, 9
    args = [rng.standard_normal((b, d, L)) for _ in range(3)] + [-rng.uniform(0.1, 2, d), rng.standard_normal((b, d))]
    ids = np.array([[0, 0, 1, 1, 1, -1, 2, -1, -1], [-1, 0, 0, 0, 3, 3, 3, 3, 4]]) if packed else None
    dy, dlast = rng.standard_normal((b, d, L)), rng.standard_normal((b, d))

    def f(*a):
        r = bo.scan(*a, ids)
        return (r["out"] * dy).sum() + (r["last"] * dlast).sum()

    r = bo.scan(*args, ids, dy, dlast)
    _difference(f, args, [r[k] for k in ("du", "dr", "di", "dA", "dh0")], rng)


@pytest.mark.parametrize("rms", [False, True])
def test_norm_oracle_gradient(rms):
    rng = np.random.default_rng(1)
    t = torch.from_numpy
    x, res, w, b = (rng.standard_normal(s) for s in ((4, 7), (4, 7), (7,), (7,)))
    dy, ds = rng.standard_normal((4, 7)), rng.standard_normal((4, 7))

    def f(x, res, w, b):
        r = bo.norm(t(x), t(w), t(b), t(res), torch.float64, rms=rms)
        return (r["out"] * dy).sum() + (r["s"] * ds).sum()

    r = bo.norm(t(x), t(w), t(b), t(res), torch.float64, rms=rms, dy=t(dy), ds=t(ds))
    _difference(f, [x, res, w, b], [r["dx"], r["dx"], r["dw"], r["db"]], rng)


@pytest.mark.parametrize("before", [False, True])
def test_gated_oracle_gradient(before):
    rng = np.random.default_rng(2)
    t = torch.from_numpy
    x, z, w = (rng.standard_normal(s) for s in ((4, 12), (4, 12), (12,)))
    dy = rng.standard_normal((4, 12))

    def f(x, z, w):
        return (bo.gated(t(x), t(z), t(w), group=4, before=before)["out"] * dy).sum()

    r = bo.gated(t(x), t(z), t(w), group=4, before=before, dy=t(dy))
    _difference(f, [x, z, w], [r["dx"], r["dz"], r["dw"]], rng)
