"""Head norms with rotation, attention with a decaying state, the loss against a teacher's top logits, at the limits of what
they are given: how often a result is rounded, values that are not finite or nearly so, and waits that run out.  Formulas,
data and calls are those of test_student_ops.py; u is half a step of a type, relative (bf16 2^-8, fp32 2^-24)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from test_student_ops import (KINDS, U, Linear, _distill_calls, _distill_data, _distill_near, _distill_ref, _form, _linear_data, _near,  # noqa: E402,F401
                              _norm_data, _norm_shape, _ok, _ptr, _stream)

gpu = pytest.mark.gpu


# ---------------------------------------------------------------- attention with a decaying state

def _linear_forms(case, t, behind, decay, n, s0, ds):
    """What out, dq, dk, dv are the form of, as arguments of _form in 64 bits, and how its results lie as rows"""
    B, H, dk, dv, T = case[:5]
    scale = dk ** -0.5
    q, k, v, do = (torch.where(behind, 0, t[x]).double().view(T, B, H, -1).permute(1, 2, 0, 3) for x in ("q", "k", "v", "dout"))
    zero = torch.zeros(B, H, dk, dv, device="cuda", dtype=torch.float64)
    s0, ds = (zero if x is None else x.double() for x in (s0, ds))
    d64 = decay.cuda().double()
    turned = lambda x: x.transpose(2, 3)  # noqa: E731
    return {"out": (q, k, v, s0, d64, n, scale, scale, 1.0, False), "dq": (do, v, k, turned(s0), d64, n, scale, scale, 1.0, False),
            "dk": (v, do, q, turned(ds), d64, n, scale, 1.0, scale, True), "dv": (k, q, do, ds, d64, n, scale, 1.0, scale, True)}


@gpu
@pytest.mark.parametrize("case", [
    (2, 2, 64, 64, 64, None, 1), (3, 2, 64, 64, 200, (200, 97, 0), 1), (150, 1, 64, 64, 100, None, 1), (2, 2, 40, 64, 333, (333, 100), 1),
    (1, 1, 64, 64, 1025, (1000,), 1), (2, 1, 128, 128, 700, (700, 333), 1), (1, 2, 32, 32, 513, None, 0), (1, 1, 16, 128, 600, None, 1),
    (1, 1, 128, 64, 200, None, 1), (13, 8, 64, 64, 50, None, 1), (2, 2, 64, 64, 6, None, 1)])
def test_linear_attention_rounds_a_bf16_result_once(pkg, case):
    """A result is off by its own rounding, u of it, and otherwise by far less: pair weights and a state's elements as factors
    keep 16 bits (2^-16 of them), the decayed values that a state adds up 16 bits too where it is no result: 2^-15 of the same sum over
    absolute values, and fp32 sums that tensor cores cut, 2^-23 a step of the longest chain."""
    kind = torch.bfloat16
    t, n, behind, decay, s0, ds, length = _linear_data(case, kind, seed=21)
    B, H, dk, dv, T = case[:5]
    op = Linear(pkg, case, kind, t, decay, s0, ds, length)
    out, _ = op.forward()
    got = {"out": out, **dict(zip(("dq", "dk", "dv"), op.backward()))}
    steps = max(dk, dv) + 64 + T / 16 + 40
    for name, form in _linear_forms(case, t, behind, decay, n, s0, ds).items():
        rows = lambda x: x.permute(2, 0, 1, 3).reshape(T * B, -1)  # noqa: E731
        want = rows(_form(*form)[0])
        size = rows(_form(*(x.abs() if isinstance(x, torch.Tensor) and x.is_floating_point() else x for x in form))[0])
        _near(got[name], want, U[kind] * want.abs() + (2.0 ** -15 + steps * 2.0 ** -23) * size + 1e-30, name)
