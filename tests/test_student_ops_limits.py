"""Head norms with rotation, attention with a decaying state, the loss against a teacher's top logits, at the limits of what
they are given: how often a result is rounded, values that are not finite or nearly so, and waits that run out.  Formulas,
data and calls are those of test_student_ops.py; u is half a step of a type, relative (bf16 2^-8, fp32 2^-24)."""
import ctypes as C
import math
import os
import subprocess

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")

from test_student_ops import (KINDS, U, Linear, _distill_calls, _distill_data, _distill_near, _distill_ref, _form, _linear_data, _near,  # noqa: E402,F401
                              _norm_data, _norm_ref, _norm_shape, _ok, _ptr, _stream)

gpu = pytest.mark.gpu


# ---------------------------------------------------------------- head norms with rotation

@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", [(5, 3, 1, 64, 64, 0, 0, 0, 1), (33, 1, 1, 32, 32, 1, 0, 0, 1), (1, 1, 1, 2, 0, 0, 0, 0, 1), (100, 7, 3, 96, 32, 0, 0, 0, 1),
                                  (3, 2, 0, 128, 64, 0, 0, 0, 1)])
def test_qk_norm_without_eps(pkg, case, kind):
    """eps 0 and rows that fill no warp, against 64 bits: nothing of lanes without a head.  Tolerances of the test with eps."""
    N, H, Hk, d, rot, adj = case[:6]
    t, gain, _ = _norm_data((min(N, 4), *case[1:]), kind)  # no padding: that takes more than four rows
    t = {n: x.repeat(N // x.shape[0] + 1, 1)[:N] for n, x in t.items()}
    assert all(x.is_contiguous() for x in t.values())
    pos = torch.arange(N, device="cuda").int()
    shape = _norm_shape(pkg, case, kind)
    shape.eps = 0.0
    lib, need = pkg.library(), C.c_size_t()
    _ok(pkg, lib.nncu_qk_norm_rope_workspace(C.byref(shape), C.byref(need)))
    room = torch.full((need.value,), 255, dtype=torch.uint8, device="cuda")
    dgain = {n: torch.full((d,), float("nan"), device="cuda") for n in "qk"}
    new, back = ({n: torch.full_like(t[n], 7.0) for n in "qk" if n in t} for _ in range(2))
    _ok(pkg, lib.nncu_qk_norm_rope_forward(C.byref(shape), _ptr(t["q"]), _ptr(t.get("k")), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos), _ptr(new["q"]),
                                           _ptr(new.get("k")), _stream()))
    _ok(pkg, lib.nncu_qk_norm_rope_backward(C.byref(shape), _ptr(t["q"]), _ptr(t.get("k")), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos), _ptr(t["dq_out"]),
                                            _ptr(t.get("dk_out")), _ptr(back["q"]), _ptr(back.get("k")), _ptr(dgain["q"]), _ptr(dgain["k"]) if Hk else None,
                                            _ptr(room), need.value, _stream()))
    f = 2.0 ** -24
    for n, h in (("q", H), ("k", Hk)):
        if not h:
            continue
        x, gn, dy = t[n].double().requires_grad_(), gain[n].double().requires_grad_(), t["d%s_out" % n].double()
        want = _norm_ref(x, gn, pos, d, rot, adj, 0.0, 10000.0)
        dx, dg = torch.autograd.grad(want, (x, gn), dy)
        spread = lambda y: y.expand(-1, -1, d).reshape(N, -1)  # noqa: E731
        size = spread(want.detach().view(N, h, d).norm(dim=-1, keepdim=True))
        _near(new[n], want.detach(), U[kind] * want.detach().abs() + 16 * f * size, n)
        up = dy.view(N, h, d).norm(dim=-1, keepdim=True)
        rs = 1 / x.detach().view(N, h, d).square().mean(-1, keepdim=True).sqrt()
        _near(back[n], dx, U[kind] * dx.abs() + (16 + d) * f * spread(up * rs * gain[n].abs().max().double()), "d" + n)
        _near(dgain[n], dg, f * (16 + math.sqrt(N * h)) * (up * math.sqrt(d)).sum(), "dgain_" + n)


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


@gpu
@pytest.mark.parametrize("B,d_key,d_value,T", [(40, 64, 64, 64), (150, 64, 64, 200), (40, 32, 32, 130), (3, 128, 128, 130), (6, 64, 64, 1024), (2, 128, 128, 700),
                                               (3, 40, 64, 333), (150, 32, 96, 90)])
def test_linear_attention_states_are_fp32_sums_of_fp32_products(pkg, B, d_key, d_value, T):
    """Each stream has one token that is not zero, in its last 60 (first 60 for the gradient): a state is that token's product times
    a power of the decay.  Off by that power (two steps, and 2^-24 of its exponent), the decayed factor's rounding, three terms'
    sums that are cut, a step for each chunk and part behind it: 16 steps of 2^-24.  Two terms of the factor would leave up to 2^-16."""
    kind = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(T + d_key)
    stream = torch.arange(B, device="cuda")
    live = T - 1 - (7 * stream + 3) % 60
    one = lambda d: torch.randn(B, d, generator=g, device="cuda").to(kind)  # noqa: E731
    k, v, q, dout = one(d_key), one(d_value), one(d_key), one(d_value)

    def rows(x, at):
        y = torch.zeros(T, B, x.shape[1], device="cuda", dtype=kind)
        y[at, stream] = x
        return y.view(T * B, -1)

    decay = torch.tensor([0.97])
    t = dict(q=rows(q, T - 1 - live), k=rows(k, live), v=rows(v, live), dout=rows(dout, T - 1 - live))
    op = Linear(pkg, (B, 1, d_key, d_value, T), kind, t, decay, None, None, None)
    _, state = op.forward()
    dstate = op.backward()[3]
    l = decay.cuda().double()
    outer = lambda a, b: a.double()[:, :, None] * b.double()[:, None, :]  # noqa: E731
    behind = (T - 1 - live)[:, None, None]
    want = l ** behind * outer(k, v)
    _near(state[:, 0], want, 16 * 2.0 ** -24 * want.abs(), "state")
    want = d_key ** -0.5 * l ** (behind + 1) * outer(q, dout)
    _near(dstate[:, 0], want, 16 * 2.0 ** -24 * want.abs(), "dstate")


@gpu
@pytest.mark.parametrize("d", [16, 64, 7])
def test_linear_attention_decays_a_token_by_the_decay_given(pkg, d):
    """One token of nothing: the state times the decay, rounded once, forward and back: no bias that calls one after the other
    would add up.  Half-lives from less than a token to half a million."""
    H = 64
    decay = (1 - 2.0 ** -torch.linspace(0.2, 19.5, H, dtype=torch.float64)).float()
    g = torch.Generator(device="cuda").manual_seed(d)
    s0, ds = (torch.randn(2, H, d, d, generator=g, device="cuda") for _ in range(2))
    nothing = torch.zeros(2, H * d, device="cuda")
    op = Linear(pkg, (2, H, d, d, 1), torch.float32, dict(q=nothing, k=nothing, v=nothing, dout=nothing), decay, s0, ds, None)
    by = decay.cuda()[None, :, None, None]
    assert torch.equal(op.forward()[1], s0 * by) and torch.equal(op.backward()[3], ds * by)
    # five tokens: five times
    five = nothing.repeat(5, 1)
    op = Linear(pkg, (2, H, d, d, 5), torch.float32, dict(q=five, k=five, v=five, dout=five), decay, s0, ds, None)
    assert torch.equal(op.forward()[1], s0 * by * by * by * by * by) and torch.equal(op.backward()[3], ds * by * by * by * by * by)


# ---------------------------------------------------------------- the loss against a teacher's top logits

def _distill_all(pkg, z, ids, top, targets, weight, tau, share, grad_kind):
    """Losses of the fused call and of the forward call, gradients of the fused call and of the pair, whatever they are"""
    lib = pkg.library()
    N, V = z.shape
    shape = pkg.abi.DistillShape(n_rows=N, n_symbols=V, n_top=ids.shape[1], ld_logits=z.stride(0), temperature=tau, teacher_share=share,
                                 logits_bf16=int(z.dtype == torch.bfloat16), grad_bf16=int(grad_kind == torch.bfloat16))
    loss, loss2, lse = (torch.full((N * k,), 7.0, device="cuda") for k in (1, 1, 2))
    dz, dz2 = (torch.full((N, V), 7.0, device="cuda", dtype=grad_kind) for _ in range(2))
    args = tuple(_ptr(x) for x in (z, ids, top, targets, weight))
    _ok(pkg, lib.nncu_distill_gradient(C.byref(shape), *args, _ptr(loss), _ptr(dz), _stream()))
    _ok(pkg, lib.nncu_distill_forward(C.byref(shape), *args, _ptr(loss2), _ptr(lse), _stream()))
    _ok(pkg, lib.nncu_distill_backward(C.byref(shape), *args, _ptr(lse), _ptr(dz2), _stream()))
    return (loss, loss2), (dz, dz2)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,V,tau,share", [(9, 300, 1.0, 0.5), (9, 300, 2.0, 1.0), (700, 5000, 3.0, 0.5), (9, 60000, 2.0, 0.5), (9, 4, 1.0, 0.0)])
def test_distillation_of_logits_that_are_not_numbers(pkg, kind, N, V, tau, share):
    """Rows of nothing but NaN, of NaN and -inf, with one NaN or +inf: NaN, not the zeros of a row without symbols; the rows
    beside them are what they are alone"""
    nan = float("nan")
    z, ids, top, targets, weight = _distill_data(N, V, 3, kind, seed=31)
    want, grad = _distill_ref(z, ids, top, targets, weight, tau, share)
    z[1] = nan
    z[2, ::2], z[2, 1::2] = -math.inf, nan
    z[3, V - 1] = nan
    z[4] = -math.inf
    z[5, V // 2] = math.inf
    z[6], weight[6] = nan, 0.0
    bad, good = [1, 2, 3, 5], [r for r in range(N) if r == 0 or r > 6]
    losses, grads = _distill_all(pkg, z, ids, top, targets, weight, tau, share, kind)
    for x in (*losses, *grads):
        assert bool(x[bad].isnan().all()), x[bad]
        assert bool((x[[4, 6]] == 0).all())
    for loss in losses:
        _distill_near(loss[good], [x[good] for x in grads], want[good], grad[good], weight[good], tau, share, kind, V)


@gpu
@pytest.mark.parametrize("V,K,bad", [(300, 20, float("nan")), (300, 20, math.inf), (9000, 300, float("nan")), (60000, 20, math.inf)])
def test_distillation_by_a_teacher_that_is_not_a_number(pkg, V, K, bad):
    """NaN or +inf among a row's entries: NaN in its loss and at the symbols they name, not a row whose teacher is not there; an
    entry that is not there may hold anything"""
    z, ids, top, targets, weight = _distill_data(7, V, K, torch.float32, seed=32)
    ids[4, 1:][ids[4, 1:] == ids[4, 0]] = -1
    top[1, 3], top[2] = bad, bad
    ids[3, 0], top[3, 0] = -1, bad
    top[4, 0] = bad
    top[5] = -math.inf
    clean = torch.where((top - top == 0) | (top == -math.inf), top, 0)
    want, grad = _distill_ref(z, torch.where((top == -math.inf).all(1, keepdim=True), -1, ids), clean, targets, weight, 2.0, 0.5)
    losses, grads = _distill_all(pkg, z, ids, top, targets, weight, 2.0, 0.5, torch.float32)
    for r in (1, 2, 4):
        named = ids[r][ids[r] >= 0].long()
        assert all(bool(x[r].isnan()) for x in losses) and all(bool(x[r, named].isnan().all()) for x in grads), r
    for loss in losses:
        _distill_near(loss[[0, 3, 5, 6]], [x[[0, 3, 5, 6]] for x in grads], want[[0, 3, 5, 6]], grad[[0, 3, 5, 6]], weight[[0, 3, 5, 6]], 2.0, 0.5, torch.float32, V)
    # of a share of 0 nothing is asked
    for x in (y for z in _distill_all(pkg, z, ids, top, targets, weight, 2.0, 0.0, torch.float32) for y in z):
        assert bool(x.isfinite().all())


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [300, 16384, 70000])
@pytest.mark.parametrize("tau", [0.01, 0.25, 8.0, 20.0, 100.0, 1e4])
def test_distillation_at_temperatures_far_from_one(pkg, kind, V, tau):
    """The pair of calls as well as the fused one, where p and p_temperature have little in common.  Tolerances of the test at
    ordinary temperatures."""
    z, ids, top, targets, weight = _distill_data(8, V, 30, kind, seed=33)
    got = _distill_calls(pkg, z, ids, top, targets, weight / tau, tau, 0.5, kind)
    want, grad = _distill_ref(z, ids, top, targets, weight / tau, tau, 0.5)
    _distill_near(got[0], got[1:], want, grad, weight / tau, tau, 0.5, kind, V)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,V,tau", [(9, 1000, 1.0), (9, 1000, 2.0), (9, 1003, 3.0), (9, 60001, 2.0), (700, 5001, 0.3)])
def test_distillation_of_logits_far_from_zero(pkg, kind, N, V, tau):
    """Rows of nothing but a type's lowest or largest value, masks of the lowest, logits about 1e4 and -3e6, in all three calls:
    a constant on a row's logits changes nothing.  Tolerances of the test at ordinary logits."""
    z, ids, top, targets, weight = _distill_data(N, V, 30, kind, seed=34)
    low, high = torch.finfo(kind).min, torch.finfo(kind).max
    half = V // 2
    z[1] = low
    z[2, half:] = low
    ids[2], targets[2] = ids[2] % half, targets[2] % half
    z[3] = (z[3].double() + 1e4).to(kind)
    z[4] = (z[4].double() - 3e6).to(kind)
    z[5] = high
    top[6] = torch.finfo(torch.float32).min
    top[7, ::2] = torch.finfo(torch.float32).min
    z[8], z[8, 17] = low, 0.5
    ids[8], targets[8] = 17, 17
    got = _distill_calls(pkg, z, ids, top, targets, weight, tau, 0.5, kind)
    want, grad = _distill_ref(z, ids, top, targets, weight, tau, 0.5)
    _distill_near(got[0], got[1:], want, grad, weight, tau, 0.5, kind, V)


@gpu
def test_distillation_by_a_teacher_who_wants_a_masked_symbol(pkg):
    """A finite mask's loss is finite: the logits' distance, to fp32's digits of it"""
    z, ids, top, targets, weight = _distill_data(4, 500, 6, torch.float32, seed=35)
    ids[1], top[1], ids[1, 0] = -1, 0.0, 7
    z[1, 7], z[2, 9], targets[2] = -3e38, -3e38, 9
    got = _distill_calls(pkg, z, ids, top, targets, weight, 1.0, 0.5, torch.float32)
    want, grad = _distill_ref(z, ids, top, targets, weight, 1.0, 0.5)
    _distill_near(got[0], got[1:], want, grad, weight, 1.0, 0.5, torch.float32, 500)


def test_distillation_refuses_temperatures_that_overflow(pkg):
    """tau^2 and 1 / tau are factors of the loss and of the logits"""
    lib, one = pkg.library(), 4096
    for tau, share, refused in ((1e20, 0.5, 1), (1e-39, 0.5, 1), (1e20, 0.0, 0), (1e-39, 0.0, 0), (1e19, 0.5, 0), (1e-37, 0.5, 0)):
        shape = pkg.abi.DistillShape(n_rows=4, n_symbols=100, n_top=5, temperature=tau, teacher_share=share)
        # an address that is no multiple of four is refused too, behind the shape: nothing is ever launched
        assert lib.nncu_distill_gradient(C.byref(shape), one + 2, one, one, None, None, one, 2 * one, None) == pkg.abi.ERR_INVALID
        assert (b"temperature" in lib.nncu_last_error()) == bool(refused), (tau, share)


# ---------------------------------------------------------------- the model's own path

def _model(pkg, bf16, V=300):
    kw = dict(n_layer=2, d_model=64, n_head=2, d_key=32, d_inner=128, d_pos=24, mem_len=16, seg_len=16, n_streams=4, n_symbols=V, use_bf16=bf16, init_range=0.2)
    m = pkg.TrfModel(pkg.abi.make_params(**kw))
    m.reset()
    return m


@gpu
@pytest.mark.parametrize("bf16", [0, 1])
def test_model_and_a_teacher_that_is_not_a_number(pkg, bf16):
    """The same of the model's loss; entries of nothing but -inf are no teacher; and the plain loss behind it is what it was"""
    np = pytest.importorskip("numpy")
    T, B, K, V = 16, 4, 40, 300
    rng = np.random.default_rng(7)
    m = _model(pkg, bf16, V)
    ids_in, tg = (rng.integers(0, V, (T, B)).astype(np.int32) for _ in range(2))
    ids = rng.integers(0, V, (T, B, K)).astype(np.int32)
    top = rng.normal(size=(T, B, K)).astype(np.float32)
    m.eval(-1, ids_in, read=False)
    plain = m.eval_gradient(tg)
    grads = {n: m.get_grad(n) for n in m.info}
    taught = m.eval_gradient_distill(tg, ids, top, 0.5)
    assert math.isfinite(taught)
    for bad in (float("nan"), math.inf):
        for k in (slice(0, 1), slice(35, 36), slice(0, K)):
            rows = top.copy()
            rows[3, 1, k] = bad
            assert math.isnan(m.eval_gradient_distill(tg, ids, rows, 0.5)), (bad, k)
            assert m.eval_gradient_distill(tg, ids, rows, 0.0) == plain
            assert all(np.array_equal(m.get_grad(n), grads[n]) for n in m.info)
            away = ids.copy()
            away[3, 1, k] = -1
            assert math.isfinite(m.eval_gradient_distill(tg, away, rows, 0.5))
    assert m.eval_gradient_distill(tg, ids, np.full_like(top, -np.inf), 0.5) == plain
    assert all(np.array_equal(m.get_grad(n), grads[n]) for n in m.info)
    assert m.eval_gradient_distill(tg, ids, top, 0.5) == taught
    assert m.eval_gradient(tg) == plain
    assert all(np.array_equal(m.get_grad(n), grads[n]) for n in m.info)
    m.close()


@gpu
@pytest.mark.parametrize("bf16", [0, 1])
def test_model_and_teachers_of_other_sizes_and_shares(pkg, bf16):
    """Entries and share change from step to step behind captured passes: 40 entries of which three are there are the bits of
    three; a share's loss lies between the target's own and the teacher's by its weight (fp32 sums of 64 rows: 2^-24 * 64)"""
    np = pytest.importorskip("numpy")
    T, B, V = 16, 4, 300
    rng = np.random.default_rng(11)
    one, two = _model(pkg, bf16, V), _model(pkg, bf16, V)
    for m in (one, two):
        for n in m.info:
            m.set_param(n, one.get_param(n))
        m._ck(m.lib.nncu_own_stream(m.h))
    for step in range(12):
        ids_in, tg = (rng.integers(0, V, (T, B)).astype(np.int32) for _ in range(2))
        ids = rng.integers(0, V, (T, B, 3)).astype(np.int32)
        top = rng.normal(size=(T, B, 3)).astype(np.float32)
        wide = np.full((T, B, 40), V, np.int32), np.full((T, B, 40), np.nan, np.float32)
        wide[0][..., :3], wide[1][..., :3] = ids, top
        share = (0.25, 0.25, 0.25, 0.75)[step % 4]
        for m in (one, two):
            m.eval(-1, ids_in, read=False)
        want = one.eval_gradient_distill(tg, ids, top, share)
        few = step % 3 == 0
        assert two.eval_gradient_distill(tg, *((ids, top) if few else wide), share) == want
        for n in one.info:
            assert np.array_equal(one.get_grad(n), two.get_grad(n)), (step, n)
        ends = [two.eval_gradient_distill(tg, ids, top, s) for s in (0.0, 1.0)]
        assert abs(want - (1 - share) * ends[0] - share * ends[1]) <= 2.0 ** -24 * 64 * (abs(ends[0]) + abs(ends[1]))
        for m in (one, two):
            assert m.eval_gradient(tg) == ends[0]
            m.update()
    one.close()
    two.close()


# ---------------------------------------------------------------- waits that run out

@pytest.fixture(scope="module")
def expired(tmp_path_factory, pkg):
    """The kernels compiled with waits that give up (tests/expired_copies.cu); expire(thread, parity) says which"""
    nvcc = pkg.loader._nvcc()
    if nvcc is None:
        pytest.skip("needs nvcc")
    out = str(tmp_path_factory.mktemp("expired") / "expired.so")
    subprocess.run([nvcc] + pkg.loader.NVCC_FLAGS + ["--split-compile=0", "-I", os.path.join(ROOT, "include"), "-I", pkg.loader.CSRC, "-o", out,
                                                     os.path.join(ROOT, "tests", "expired_copies.cu")], check=True, capture_output=True)
    lib = C.CDLL(out)
    lib.nncu_last_error.restype = C.c_char_p
    yield lib
    lib.expire(0, 2)


@gpu
@pytest.mark.parametrize("slots,late", [(1, 0), (2, 0), (3, 1), (4, 1)])
@pytest.mark.parametrize("thread,parity", [(-1, -1), (-1, 1), (0, 1), (70, 0), (127, 1)])
def test_expired_waits_of_distillation_leave_no_result(pkg, expired, slots, late, thread, parity):
    """Rows of 3 CTAs, row 3 n + c the n-th of CTA c, whose copy completes a phase of parity n / slots: from the first one that a
    thread did not see arrive, all that a CTA owes is NaN, those before it are as they are otherwise"""
    N, V, K, ctas = 40, 1003, 5, 3
    z, ids, top, targets, _ = _distill_data(N, V, K, torch.float32, seed=41)
    z[:, V // 2] += 1.0

    def run(what, *results):
        rc = expired.expired_distill(what, late, ctas, slots, N, V, K, *(C.c_void_p(_ptr(x)) for x in (z, ids, top, targets, *results)))
        assert rc == 0, expired.nncu_last_error()

    def all_calls(lse=None):
        loss, loss2, dz, dz2 = (torch.ones(n, device="cuda") for n in (N, N, N * V, N * V))
        sums = torch.ones(2 * N, device="cuda")
        run(1, loss, sums, None)
        run(2, None, sums if lse is None else lse, dz)
        run(3, loss2, None, dz2)
        torch.cuda.synchronize()
        return loss, sums.view(N, 2), dz.view(N, V), loss2, dz2.view(N, V)

    assert expired.expire(0, 2) == 0
    want = all_calls()
    assert all(bool(x.isfinite().all()) for x in want)
    assert expired.expire(thread, parity) == 0
    got = all_calls(want[1])
    gone = torch.arange(N, device="cuda") // ctas >= (slots if parity == 1 else 0)
    assert bool(gone.any())
    for x, y in zip(got, want):
        assert bool(x[gone].isnan().all()) and torch.equal(x[~gone], y[~gone])
    assert expired.expire(0, 2) == 0
    assert all(torch.equal(x, y) for x, y in zip(all_calls(), want))


class _Library:
    """The package with another library for its calls"""

    def __init__(self, pkg, lib):
        self.abi, self.lib = pkg.abi, lib
        for name in ("nncu_linear_attention_workspace", "nncu_linear_attention_forward", "nncu_linear_attention_backward"):
            call = getattr(lib, name)
            call.restype, call.argtypes = pkg.abi.PROTOTYPES[name]

    def library(self):
        return self.lib


@gpu
@pytest.mark.parametrize("thread,parity", [(-1, -1), (-1, 0), (-1, 1), (0, 1), (70, 1), (255, 1), (130, 0)])
def test_expired_waits_of_linear_attention_leave_no_result(pkg, expired, thread, parity):
    """150 streams of five chunks, k-th from the end for dk and dv: chunk k's copy completes a phase of parity k / 2, the second left
    factor's (dk) one of parity k.  What a CTA owes is NaN from the first chunk on that a thread did not see arrive, states
    among it; in a chunk that misses the second left factor alone, the dk of that thread's sixteen rows."""
    case = (150, 1, 64, 64, 300, None, 1)
    B, H, d, _, T = case[:5]
    t, n, behind, decay, s0, ds, length = _linear_data(case, torch.bfloat16, seed=42)
    op = Linear(_Library(pkg, expired), case, torch.bfloat16, t, decay, s0, ds, length)
    call = lambda: [x.clone() for x in (*op.forward(), *op.backward())]  # noqa: E731
    assert expired.expire(0, 2) == 0
    want = call()
    assert all(bool(x.isfinite().all()) for x in want)
    assert expired.expire(thread, parity) == 0
    got = call()
    torch.cuda.synchronize()
    first = 2 if parity == 1 else 0
    at = torch.arange(T, device="cuda")
    for name, x, y in zip(("out", "state", "dq", "dk", "dv", "dstate"), got, want):
        if "state" in name:
            assert bool(x.isnan().all()), name
            continue
        x, y = x.view(T, -1), y.view(T, -1)
        chunk = (at if name in ("out", "dq") else T - 1 - at) // 64
        gone, sure = chunk >= first, chunk < first - (name == "dk")
        assert bool(x[gone].isnan().all()) and torch.equal(x[sure], y[sure]), name
        part, whole = x[~gone & ~sure].isnan(), (x == y)[~gone & ~sure]
        assert bool((part | whole).all()) and (first == 0 or name != "dk" or part.sum() == (64 if thread < 0 else 16) * B * d), name
    assert expired.expire(0, 2) == 0
    assert all(torch.equal(x, y) for x, y in zip(call(), want))


@gpu
def test_expired_waits_of_linear_attention_in_parts_leave_no_result(pkg, expired):
    """One long stream in several parts, whose sums a first pass makes"""
    case = (1, 1, 64, 64, 2560, None, 1)
    t, n, behind, decay, s0, ds, length = _linear_data(case, torch.bfloat16, seed=43)
    op = Linear(_Library(pkg, expired), case, torch.bfloat16, t, decay, s0, ds, length)
    assert op.need > 0 and expired.expire(-1, -1) == 0
    assert all(bool(x.isnan().all()) for x in (*op.forward(), *op.backward()))
    assert expired.expire(0, 2) == 0
    assert all(bool(x.isfinite().all()) for x in (*op.forward(), *op.backward()))
