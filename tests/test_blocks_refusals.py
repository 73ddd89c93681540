"""CPU tier: what refil_amd.blocks and the C entries underneath refuse, before any launch (the C checks are host code: the product library
answers them without a GPU; the shape checks of the Python layer run on the emulator's host tensors)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

import emu_util
from refil_amd import _lib, blocks

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 4)
    for call in (lambda: blocks.linrec_forward(x, x, x, x[0, 0]), lambda: blocks.linear_recurrence(x, x, x, x[0, 0]), lambda: blocks.linrec_step(x[0], x[0], x[0], x[0, 0], x[0]),
                 lambda: blocks.norm_gate_forward(x), lambda: blocks.norm_gate_residual(x), lambda: blocks.gated_ff_forward(x, x[0], x[0]), lambda: blocks.gated_ff(x, x[0], x[0])):
        with pytest.raises(ValueError, match="no host path"):
            call()


@pytest.fixture
def host(monkeypatch):
    """past the GPU guard: every refusal below comes before a launch"""
    monkeypatch.setattr(blocks, "_require_gpu", lambda t, who: None)

    def no_launch(*a):
        raise AssertionError("a refused call was launched")
    monkeypatch.setattr(blocks, "_launch", no_launch)
    with emu_util.active():
        yield


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("error,needle,call", [
    (TypeError, "dtype torch.float64", lambda: blocks.linrec_forward(*[z(2, 3, 4, dtype=torch.float64)] * 3, z(4))),
    (ValueError, "expected \\[B, T, D\\]", lambda: blocks.linrec_forward(*[z(3, 4)] * 3, z(4))),
    (TypeError, "decay_gate is torch.bfloat16", lambda: blocks.linrec_forward(z(2, 3, 4), z(2, 3, 4, dtype=torch.bfloat16), z(2, 3, 4), z(4))),
    (ValueError, "input_gate has shape", lambda: blocks.linrec_forward(z(2, 3, 4), z(2, 3, 4), z(2, 3, 5), z(4))),
    (ValueError, "decay has shape", lambda: blocks.linrec_forward(*[z(2, 3, 4)] * 3, z(12))),
    (TypeError, "decay is torch.float16", lambda: blocks.linrec_forward(*[z(2, 3, 4)] * 3, z(4, dtype=torch.float16))),
    (TypeError, "h0 is torch.bfloat16", lambda: blocks.linrec_forward(*[z(2, 3, 4)] * 3, z(4), h0=z(2, 4, dtype=torch.bfloat16))),
    (ValueError, "h0 has shape", lambda: blocks.linrec_forward(*[z(2, 3, 5, 4)] * 3, z(4), h0=z(2, 4))),
    (TypeError, "reset is torch.float32", lambda: blocks.linrec_forward(*[z(2, 3, 4)] * 3, z(4), reset=z(2, 3))),
    (ValueError, "lengths must be", lambda: blocks.linrec_forward(*[z(2, 3, 4)] * 3, z(4), lengths=z(2))),
    (ValueError, "D must be positive", lambda: blocks.linrec_forward(*[z(2, 3, 0)] * 3, z(0))),
    (ValueError, "saved has shape", lambda: blocks.linrec_backward(*[z(2, 70, 4)] * 4, z(4), z(2 * 4))),
    (ValueError, "state must be", lambda: blocks.linrec_step(*[z(2, 4)] * 3, z(4), z(3, 5))),
    (ValueError, "state must be", lambda: blocks.linrec_step(*[z(2, 4)] * 3, z(4), z(4, 3).t())),
    (ValueError, "2 rows, 1 states", lambda: blocks.linrec_step(*[z(2, 4)] * 3, z(4), z(1, 4))),
    (ValueError, "slots must be", lambda: blocks.linrec_step(*[z(2, 4)] * 3, z(4), z(3, 4), slots=torch.zeros(2, dtype=torch.int64))),
    (ValueError, "overlaps", lambda: (lambda s: blocks.linrec_step(*[z(2, 4)] * 3, z(4), s[:3], state_out=s[1:4]))(z(4, 4))),
    (ValueError, "needs the block's output", lambda: blocks.norm_gate_forward(z(2, 4), None, z(2, 4))),
    (ValueError, "post_weight has shape", lambda: blocks.norm_gate_forward(z(2, 4), z(2, 4), post_weight=z(5))),
    (ValueError, "eps must be positive", lambda: blocks.norm_gate_forward(z(2, 4), eps=0.0)),
    (ValueError, "neither y nor n", lambda: blocks.norm_gate_forward(z(2, 4), want_y=False, want_n=False)),
    (ValueError, "neither dy nor dn", lambda: blocks.norm_gate_backward(None, None, z(2, 4))),
    (ValueError, "row_mask has shape", lambda: blocks.norm_gate_forward(z(2, 4), row_mask=torch.zeros(2, 4, dtype=torch.bool))),
    (ValueError, "act 'relu'", lambda: blocks.gated_ff_forward(z(2, 4), z(3, 4), z(3, 4), act="relu")),
    (ValueError, "expected \\[..., D\\] and \\[F, D\\]", lambda: blocks.gated_ff_forward(z(2, 5), z(3, 4), z(3, 4))),
    (ValueError, "w_up has shape", lambda: blocks.gated_ff_forward(z(2, 4), z(3, 4), z(2, 4))),
    (TypeError, "w_gate is torch.bfloat16", lambda: blocks.gated_ff_forward(z(2, 4), z(3, 4, dtype=torch.bfloat16), z(3, 4))),
    (ValueError, "b_up has shape", lambda: blocks.gated_ff_forward(z(2, 4), z(3, 4), z(3, 4), None, z(4))),
    (ValueError, "saved has shape", lambda: blocks.gated_ff_backward(z(2, 3), z(2, 4), z(3, 4), z(3, 4), z(2, 2, 4))),
    (ValueError, "dh has shape", lambda: blocks.gated_ff_backward(z(2, 4), z(2, 4), z(3, 4), z(3, 4), z(2, 2, 3))),
])
def test_bad_arguments_are_refused_before_a_launch(host, error, needle, call):
    with pytest.raises(error, match=needle):
        call()


def _err():
    return _lib.lib().refil_last_error().decode()


def test_c_entries_refuse():
    """every C entry names what is wrong and launches nothing (pointers here are host addresses nobody reads)"""
    L = _lib.lib()
    buf = (C.c_float * 64)()
    p = C.addressof(buf)
    for fn, what in ((L.refil_linrec_forward, "refil_linrec_forward"), (L.refil_linrec_backward, "refil_linrec_backward"), (L.refil_linrec_step, "refil_linrec_step"),
                     (L.refil_norm_gate_forward, "refil_norm_gate_forward"), (L.refil_norm_gate_backward, "refil_norm_gate_backward"),
                     (L.refil_gated_ff_forward, "refil_gated_ff_forward"), (L.refil_gated_ff_backward, "refil_gated_ff_backward")):
        assert fn(None, None) != 0 and f"{what}: null desc" in _err()

    def rec(**kw):
        d = _lib.LinrecDesc(x=p, ga=p, gi=p, decay=p, y=p, B=1, T=2, C=4, D=4, scale=8.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    for kw, needle in ((dict(dtype=3), "dtype 3"), (dict(D=3), "multiple of D 3"), (dict(D=0), "D 0 positive"), (dict(B=-1), "B -1"), (dict(x=None), "x, ga, gi and y"),
                       (dict(decay=None), "decay is NULL"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")):
        assert L.refil_linrec_forward(C.byref(rec(**kw)), None) != 0 and needle in _err(), (kw, _err())
    assert L.refil_linrec_backward(C.byref(rec()), None) != 0 and "ddecay" in _err()
    assert L.refil_linrec_backward(C.byref(rec(ddecay=p)), None) != 0 and "saved" in _err()
    assert L.refil_linrec_backward(C.byref(rec(ddecay=p, dy=p, dx=p, dga=p, dgi=p, saved=p)), None) != 0 and "workspace of 0 bytes" in _err()
    s = _lib.LinrecStepDesc(x=p, ga=p, gi=p, decay=p, state=p, state_out=p, y=p, B=2, C=4, D=4, n_slots=1, scale=8.0)
    assert L.refil_linrec_step(C.byref(s), None) != 0 and "1 state rows for 2 rows" in _err()
    s.n_slots, s.state = 2, None
    assert L.refil_linrec_step(C.byref(s), None) != 0 and "state_out and y are required" in _err()

    def norm(**kw):
        d = _lib.NormGateDesc(x=p, y=p, n=p, N=2, D=4, x_stride=4, y_stride=4, n_stride=4, alpha=1.0, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    for kw, needle in ((dict(dtype=-1), "dtype -1"), (dict(D=16385), "D 16385 in 1"), (dict(N=-1), "N -1"), (dict(eps=0.0), "eps"), (dict(gate=p), "gate needs"),
                       (dict(y=None, n=None), "neither y nor n"), (dict(x=None), "x is required")):
        assert L.refil_norm_gate_forward(C.byref(norm(**kw)), None) != 0 and needle in _err(), (kw, _err())
    assert L.refil_norm_gate_backward(C.byref(norm()), None) != 0 and "one of dy, dn" in _err()
    assert L.refil_norm_gate_backward(C.byref(norm(o=p, dy=p, dx=p)), None) != 0 and "d_o is required" in _err()
    assert L.refil_norm_gate_backward(C.byref(norm(o=p, gate=p, dy=p, dx=p, d_o=p)), None) != 0 and "dgate is required" in _err()
    assert L.refil_norm_gate_backward(C.byref(norm(dy=p, dx=p)), None) != 0 and "workspace of 0 bytes" in _err()

    def ff(**kw):
        d = _lib.GatedFfDesc(x=p, w_gate=p, w_up=p, h=p, x_stride=4, w_stride=4, h_stride=4, N=2, D=4, F=4)
        for k, v in kw.items():
            setattr(d, k, v)
        return d
    for kw, needle in ((dict(dtype=7), "dtype 7"), (dict(act=2), "act 2"), (dict(F=0), "F 0"), (dict(w_stride=3), "w_stride 3 below"), (dict(x_stride=3), "x_stride 3 below"), (dict(h=None), "h are required")):
        assert L.refil_gated_ff_forward(C.byref(ff(**kw)), None) != 0 and needle in _err(), (kw, _err())
    assert L.refil_gated_ff_backward(C.byref(ff(N=0)), None) != 0 and "no rows" in _err()
    assert L.refil_gated_ff_backward(C.byref(ff()), None) != 0 and "saved" in _err()
    assert L.refil_gated_ff_backward(C.byref(ff(saved=p, dh=p, dx=p, dw_gate=p, dw_up=p)), None) != 0 and "workspace of 0 bytes" in _err()


def test_descriptor_sizes_match_the_header():
    src = '#include "refil_hip.h"\n#include <stdio.h>\nint main(){printf("%zu %zu %zu %zu\\n",sizeof(refil_linrec_desc),sizeof(refil_linrec_step_desc),' \
          'sizeof(refil_norm_gate_desc),sizeof(refil_gated_ff_desc));return 0;}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "s.c"), os.path.join(td, "s")
        with open(c, "w") as fh:
            fh.write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        sizes = [int(v) for v in subprocess.check_output([exe]).split()]
    assert sizes == [C.sizeof(t) for t in (_lib.LinrecDesc, _lib.LinrecStepDesc, _lib.NormGateDesc, _lib.GatedFfDesc)]


def test_sizing_queries_answer_zero_for_bad_descriptors():
    L = _lib.lib()
    assert L.refil_linrec_workspace_bytes(C.byref(_lib.LinrecDesc(B=1, T=1, C=4, D=3, scale=1.0)), 1) == 0
    assert L.refil_linrec_saved_floats(C.byref(_lib.LinrecDesc(B=2, T=65, C=4, D=4, scale=1.0))) >= 2 * 2 * 4
    assert L.refil_norm_gate_workspace_bytes(C.byref(_lib.NormGateDesc(N=1, D=0, eps=1.0))) == 0
    assert L.refil_gated_ff_workspace_bytes(C.byref(_lib.GatedFfDesc(N=1, D=4, F=0)), 0) == 0


def test_gated_ff_workspace_begins_on_16_bytes():
    """its copies to LDS take 16 bytes at a time; the call before the one that is refused gets past this check, to the size's"""
    L = _lib.lib()
    buf = (C.c_float * 64)()
    p = C.addressof(buf)
    d = _lib.GatedFfDesc(x=p, w_gate=p, w_up=p, x_stride=8, w_stride=8, N=2, D=8, F=8, dtype=_lib.BF16, saved=p, dh=p, dh_stride=8, dx=p, dx_stride=8, dw_gate=p, dw_up=p)
    need = L.refil_gated_ff_workspace_bytes(C.byref(d), 1)
    base = (p + 63) // 64 * 64
    d.workspace, d.workspace_bytes = base, need - 1
    assert L.refil_gated_ff_backward(C.byref(d), None) != 0 and f"workspace of {need - 1} bytes" in _err()
    for off in (1, 4, 8):
        d.workspace, d.workspace_bytes = base + off, need
        assert L.refil_gated_ff_backward(C.byref(d), None) != 0 and "workspace must begin on 16 bytes" in _err()
