"""Head norms with rotation, attention with a decaying state, the loss against a teacher's top logits: refusals
without a GPU, and on one every form against 64 bits at the sizes and masks where it can go wrong.

Tolerances.  u is half a step of a type, relative (bf16 2^-8, fp32 2^-24).  A result of products is off by its own
rounding, u |y|, by one rounding to the operands' type of each weight that stands for a pair of rows or for a state's
element, u_in times the same sum over absolute values, and by fp32 sums: tensor cores cut instead of rounding, 2^-23
a step, for the longest chain of steps, times the same."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
KINDS = [torch.bfloat16, torch.float32]


def _ptr(x):
    return None if x is None else x.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ok(pkg, rc):
    assert rc == 0, pkg.library().nncu_last_error()


def _near(got, want, tol, what=""):
    """|got - want| <= tol element by element, NaN nowhere"""
    err = (got.double() - want).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert bool((err <= tol).all()), (what, "worst excess", worst, "largest error", err.max().item())


def _padded(shape, kind, g, pitch, scale=1.0):
    """rows in a buffer of wider rows whose other columns are NaN: (view, pitch)"""
    rows, cols = shape
    buf = torch.full((rows, pitch), float("nan"), device="cuda", dtype=kind)
    buf[:, :cols] = (scale * torch.randn(rows, cols, generator=g, device="cuda")).to(kind)
    return buf[:, :cols]


# ---------------------------------------------------------------- refusals (no GPU needed)

def _refused(pkg, rc, code=None):
    assert rc == (pkg.abi.ERR_INVALID if code is None else code)
    assert pkg.library().nncu_last_error() != b""


def test_qk_norm_refuses_bad_arguments(pkg):
    lib, one = pkg.library(), 4096
    good = dict(n_rows=4, n_head=2, n_head_k=1, d_key=8, d_rot=4, eps=1e-6, rope_base=1e4, dtype_bf16=1)

    def forward(pos=one, q=one, q_out=2 * one, k=one, k_out=3 * one, **over):
        return lib.nncu_qk_norm_rope_forward(C.byref(pkg.abi.QkNormShape(**{**good, **over})), q, k, None, None, pos, q_out, k_out, None)

    for over in (dict(n_rows=0), dict(n_head=0), dict(n_head_k=-1), dict(d_key=7), dict(d_key=0), dict(d_rot=3), dict(d_rot=10), dict(eps=-1.0),
                 dict(eps=float("nan")), dict(rope_base=0.0), dict(rope_base=float("inf")), dict(ld_q=15), dict(ld_k=7), dict(ld_q_out=8),
                 dict(ld_k_out=1), dict(pos=None), dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(q=one + 1),
                 dict(pos=one + 2), dict(q_out=one, ld_q_out=32), dict(k_out=2 * one)):
        _refused(pkg, forward(**over))
    _refused(pkg, forward(d_key=258, d_rot=0), pkg.abi.ERR_RANGE)
    assert lib.nncu_qk_norm_rope_forward(None, one, one, None, None, one, one, one, None) == pkg.abi.ERR_INVALID
    shape, need = pkg.abi.QkNormShape(**good), C.c_size_t()
    assert lib.nncu_qk_norm_rope_workspace(C.byref(shape), C.byref(need)) == 0 and need.value >= 4 * 2 * 8
    _refused(pkg, lib.nncu_qk_norm_rope_workspace(C.byref(shape), None))

    def backward(gain=one, dgain=one, room=one, n=need.value, dq=5 * one, dk=6 * one, dq_out=one):
        return lib.nncu_qk_norm_rope_backward(C.byref(shape), one, one, gain, gain, one, dq_out, one, dq, dk, dgain, dgain, room, n, None)

    for over in (dict(gain=None), dict(room=None), dict(n=need.value - 1), dict(room=one + 4), dict(dq=None), dict(dk=5 * one), dict(dq_out=None)):
        _refused(pkg, backward(**over))


def test_qk_norm_refuses_results_over_the_other_input(pkg):
    lib, a, b, c, d = pkg.library(), 4096, 8192, 12288, 16384
    s = pkg.abi.QkNormShape(n_rows=4, n_head=1, n_head_k=1, d_key=8, d_rot=0, eps=1e-6, dtype_bf16=1)
    for q_out, k_out in ((b, c), (c, a), (c, c)):
        _refused(pkg, lib.nncu_qk_norm_rope_forward(C.byref(s), a, b, None, None, None, q_out, k_out, None))
    for dq, dk in ((b, 5 * a), (5 * a, a), (d, 5 * a), (5 * a, c), (5 * a, 5 * a)):  # dq_out at c, dk_out at d
        _refused(pkg, lib.nncu_qk_norm_rope_backward(C.byref(s), a, b, None, None, None, c, d, dq, dk, None, None, None, 0, None))
    # a gain of keys that are not there
    one = pkg.abi.QkNormShape(n_rows=4, n_head=1, n_head_k=0, d_key=8, d_rot=0, eps=1e-6, dtype_bf16=1)
    _refused(pkg, lib.nncu_qk_norm_rope_backward(C.byref(one), a, None, a, a, None, c, None, d, None, a, a, a, 1 << 20, None))


def test_linear_attention_refuses_states_that_overlap(pkg):
    lib, one = pkg.library(), 1 << 20
    s = pkg.abi.LinearAttnShape(n_streams=2, n_head=1, d_key=16, d_value=16, seg_len=4, scale=1.0, dtype_bf16=1)
    d, size = (C.c_float * 1)(0.5), 2 * 16 * 16 * 4
    for off in (4, size - 4, -4):
        _refused(pkg, lib.nncu_linear_attention_forward(C.byref(s), one, one, one, d, None, 2 * one, 3 * one, 2 * one + off, None, 0, None))
        _refused(pkg, lib.nncu_linear_attention_backward(C.byref(s), one, one, one, d, None, None, 3 * one, 2 * one, 4 * one, 5 * one, 6 * one,
                                                         2 * one + off, None, 0, None))
    # the state that dq reads is not a place for dstate_in
    _refused(pkg, lib.nncu_linear_attention_backward(C.byref(s), one, one, one, d, None, 2 * one, 3 * one, None, 4 * one, 5 * one, 6 * one,
                                                     2 * one, None, 0, None))


def test_linear_attention_refuses_bad_arguments(pkg):
    lib, one = pkg.library(), 4096
    good = dict(n_streams=2, n_head=2, d_key=16, d_value=16, seg_len=4096, scale=0.25, dtype_bf16=1)
    need = C.c_size_t()
    shape = pkg.abi.LinearAttnShape(**good)
    assert lib.nncu_linear_attention_workspace(C.byref(shape), 0, C.byref(need)) == 0 and need.value > 0
    _refused(pkg, lib.nncu_linear_attention_workspace(C.byref(shape), 0, None))
    token = pkg.abi.LinearAttnShape(**{**good, "seg_len": 1})
    none = C.c_size_t(7)
    assert lib.nncu_linear_attention_workspace(C.byref(token), 1, C.byref(none)) == 0 and none.value == 0

    def forward(decay=(0.5, 1.0), q=one, k=one, v=one, out=2 * one, room=one, n=need.value, state_in=None, **over):
        d = None if decay is None else (C.c_float * len(decay))(*decay)
        return lib.nncu_linear_attention_forward(C.byref(pkg.abi.LinearAttnShape(**{**good, **over})), q, k, v, d, None, state_in, out, None, room,
                                                 n, None)

    def backward(dq=3 * one, dk=4 * one, dv=5 * one, dout=6 * one, room=one):
        d = (C.c_float * 2)(0.5, 0.5)
        return lib.nncu_linear_attention_backward(C.byref(shape), one, one, one, d, None, None, dout, None, dq, dk, dv, None, room, need.value, None)

    for over in (dict(n_streams=0), dict(n_head=0), dict(d_key=0), dict(d_value=0), dict(seg_len=0), dict(scale=float("nan")), dict(ld_q=31),
                 dict(ld_k=1), dict(ld_v=16), dict(ld_out=31), dict(decay=None), dict(decay=(0.0, 0.5)), dict(decay=(0.5, 1.5)),
                 dict(decay=(float("nan"), 1.0)), dict(decay=(-0.5, 1.0)), dict(q=None), dict(out=None), dict(out=one), dict(room=None),
                 dict(room=one + 8), dict(n=need.value - 1), dict(q=one + 1), dict(state_in=one + 2)):
        _refused(pkg, forward(**over))
    for over in (dict(d_key=129), dict(d_value=130), dict(n_head=65, decay=(0.5,) * 65), dict(seg_len=2 ** 31 - 1)):
        _refused(pkg, forward(**over), pkg.abi.ERR_RANGE)
    for over in (dict(dq=None), dict(dk=3 * one), dict(dv=one), dict(dq=6 * one), dict(dout=None), dict(room=None)):
        _refused(pkg, backward(**over))


def test_distillation_refuses_bad_arguments(pkg):
    lib, one = pkg.library(), 4096
    good = dict(n_rows=4, n_symbols=100, n_top=5, temperature=2.0, teacher_share=0.5, logits_bf16=0, grad_bf16=0)

    def gradient(z=one, ids=one, top=one, loss=one, dz=2 * one, **over):
        return lib.nncu_distill_gradient(C.byref(pkg.abi.DistillShape(**{**good, **over})), z, ids, top, None, None, loss, dz, None)

    for over in (dict(n_rows=0), dict(n_symbols=0), dict(n_top=-1), dict(temperature=0.0), dict(temperature=float("nan")),
                 dict(temperature=float("inf")), dict(teacher_share=-0.1), dict(teacher_share=1.1), dict(teacher_share=float("nan")),
                 dict(ld_logits=99), dict(ld_dlogits=1), dict(z=None), dict(ids=None), dict(top=None), dict(loss=None), dict(dz=None),
                 dict(dz=one), dict(z=one + 2), dict(ids=one + 1)):
        _refused(pkg, gradient(**over))
    _refused(pkg, gradient(n_top=1025), pkg.abi.ERR_RANGE)
    shape = pkg.abi.DistillShape(**good)
    _refused(pkg, lib.nncu_distill_forward(C.byref(shape), one, one, one, None, None, one, None, None))
    _refused(pkg, lib.nncu_distill_backward(C.byref(shape), one, one, one, None, None, None, one, None))
    assert lib.nncu_distill_gradient(None, one, one, one, None, None, one, 2 * one, None) == pkg.abi.ERR_INVALID


def test_shapes_have_the_layout_of_the_header(pkg):
    assert C.sizeof(pkg.abi.QkNormShape) == 4 * 13
    assert C.sizeof(pkg.abi.LinearAttnShape) == 4 * 11
    assert C.sizeof(pkg.abi.DistillShape) == 4 * 9


def test_student_operators_without_a_device(pkg):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib, one = pkg.library(), 4096
    s = pkg.abi.DistillShape(n_rows=1, n_symbols=2, n_top=0, temperature=1.0)
    assert lib.nncu_distill_gradient(C.byref(s), one, None, None, None, None, one, 2 * one, None) == pkg.abi.ERR_CUDA


@gpu
def test_host_memory_is_refused(pkg):
    lib = pkg.library()
    here, there = torch.zeros(64, device="cuda"), torch.zeros(64)
    s = pkg.abi.DistillShape(n_rows=1, n_symbols=8, n_top=0, temperature=1.0)
    _refused(pkg, lib.nncu_distill_gradient(C.byref(s), there.data_ptr(), None, None, None, None, here.data_ptr(), here.data_ptr() + 64, None))
    n = pkg.abi.QkNormShape(n_rows=2, n_head=1, d_key=8)
    _refused(pkg, lib.nncu_qk_norm_rope_forward(C.byref(n), here.data_ptr(), None, None, None, None, there.data_ptr(), None, None))
    a, d = pkg.abi.LinearAttnShape(n_streams=1, n_head=1, d_key=8, d_value=8, seg_len=1, scale=1.0), (C.c_float * 1)(0.5)
    p = here.data_ptr()
    _refused(pkg, lib.nncu_linear_attention_forward(C.byref(a), p, p + 32, p + 64, d, None, there.data_ptr(), p + 96, None, None, 0, None))


# ---------------------------------------------------------------- head norms with rotation

def _norm_ref(x, gain, pos, d, rot, adjacent, eps, base):
    """64 bits, pairs as complex numbers; padding rows are zeros"""
    N = x.shape[0]
    x = x.double().view(N, -1, d)
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    if gain is not None:
        n = n * gain.double()
    if rot:
        i = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64)
        ang = pos.double()[:, None, None] * base ** (-i / rot)
        z = n[..., :rot]
        z = torch.complex(z[..., 0::2], z[..., 1::2]) if adjacent else torch.complex(z[..., :rot // 2], z[..., rot // 2:])
        z = z * torch.polar(torch.ones_like(ang), ang)
        z = torch.stack((z.real, z.imag), -1).flatten(-2) if adjacent else torch.cat((z.real, z.imag), -1)
        n = torch.cat((z, n[..., rot:]), -1)
    return n.reshape(N, -1)


NORM_CASES = [  # rows, heads, key heads, d, rot, adjacent, first position, pitch beyond the row, gains
    (1, 1, 0, 2, 2, 0, 0, 0, 1), (5, 3, 1, 64, 64, 0, 7, 0, 1), (650, 8, 2, 64, 32, 1, 2 ** 30, 0, 1), (33, 2, 2, 32, 0, 0, 0, 0, 1),
    (17, 5, 3, 6, 4, 0, 1000, 0, 1), (9, 2, 1, 96, 96, 1, 12345, 8, 1), (40, 16, 16, 128, 64, 0, 2 ** 31 - 64, 16, 0), (12, 1, 1, 112, 56, 0, 3, 1, 1),
    (2000, 4, 4, 16, 16, 0, 0, 0, 1), (3, 1, 1, 256, 256, 0, 77, 0, 1), (70, 7, 7, 34, 34, 1, 5, 0, 1)]


def _norm_data(case, kind, seed=1):
    N, H, Hk, d, rot, adj, first, more, gains = case
    g = torch.Generator(device="cuda").manual_seed(seed + N)
    t = {n: _padded((N, h * d), kind, g, h * d + more) for n, h in (("q", H), ("dq_out", H), ("k", Hk), ("dk_out", Hk)) if h}
    gain = {n: 1 + 0.3 * torch.randn(d, generator=g, device="cuda") if gains else None for n in "qk"}
    pos = (first + torch.arange(N, device="cuda")).int()
    if N > 4:  # padding, NaN in it
        pos[torch.rand(N, generator=g, device="cuda") < 0.2] = -3
        for x in t.values():
            x[pos < 0] = float("nan")
    return t, gain, pos


def _norm_shape(pkg, case, kind):
    N, H, Hk, d, rot, adj, first, more, gains = case
    return pkg.abi.QkNormShape(n_rows=N, n_head=H, n_head_k=Hk, d_key=d, d_rot=rot, ld_q=H * d + more, ld_k=Hk * d + more, ld_q_out=H * d + more,
                               ld_k_out=Hk * d + more, adjacent=adj, eps=1e-6, rope_base=10000.0, dtype_bf16=int(kind == torch.bfloat16))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", NORM_CASES)
def test_qk_norm_rope_against_64_bits(pkg, case, kind):
    """Forward and backward.  A result is a sum of two normed values, off by a few fp32 roundings of each (mean, root,
    gain, sine: 16 taken) and by angles that 64 bits hold to 2^31 * 2^-52 of a turn and more; a gradient has d more terms."""
    lib = pkg.library()
    N, H, Hk, d, rot, adj, first, more, gains = case
    t, gain, pos = _norm_data(case, kind)
    shape = _norm_shape(pkg, case, kind)
    new = {n: torch.full((N, x.stride(0)), 7.0, device="cuda", dtype=kind)[:, :x.shape[1]] for n, x in t.items()}
    q, k = t["q"], t.get("k")
    _ok(pkg, lib.nncu_qk_norm_rope_forward(C.byref(shape), _ptr(q), _ptr(k), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos), _ptr(new["q"]),
                                           _ptr(new.get("k")), _stream()))
    back = {n: torch.full((N, x.stride(0)), 7.0, device="cuda", dtype=kind)[:, :x.shape[1]] for n, x in t.items()}
    dgain = {n: torch.full((d,), float("nan"), device="cuda") for n in "qk"}
    need = C.c_size_t()
    _ok(pkg, lib.nncu_qk_norm_rope_workspace(C.byref(shape), C.byref(need)))
    room = torch.full((need.value,), 255, dtype=torch.uint8, device="cuda")
    wanted = bool(gains)
    _ok(pkg, lib.nncu_qk_norm_rope_backward(C.byref(shape), _ptr(q), _ptr(k), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos), _ptr(t["dq_out"]),
                                            _ptr(t.get("dk_out")), _ptr(back["q"]), _ptr(back.get("k")), _ptr(dgain["q"]) if wanted else None,
                                            _ptr(dgain["k"]) if wanted and Hk else None, _ptr(room), need.value, _stream()))
    live = (pos >= 0)[:, None]
    u, f = U[kind], 2.0 ** -24
    turn = 2 * math.pi * 2.0 ** 31 * 2.0 ** -52
    for n, h in (("q", H), ("k", Hk)):
        if not h:
            continue
        x = torch.where(live, t[n], 0).double().requires_grad_()
        gn = None if gain[n] is None else gain[n].double().requires_grad_()
        want = torch.where(live, _norm_ref(x, gn, pos, d, rot, adj, 1e-6, 10000.0), 0)
        size = want.detach().view(N, h, d).norm(dim=-1, keepdim=True).expand(-1, -1, d).reshape(N, -1)
        _near(new[n], want.detach(), u * want.detach().abs() + (16 * f + turn) * size, n)
        dy = torch.where(live, t["d%s_out" % n], 0).double()
        grads = torch.autograd.grad(want, (x,) if gn is None else (x, gn), dy)
        rs = 1 / (x.detach().view(N, h, d).square().mean(-1, keepdim=True) + 1e-6).sqrt()
        up = dy.view(N, h, d).norm(dim=-1, keepdim=True) * (1 if gain[n] is None else gain[n].abs().max().double())
        bound = (up * rs).expand(-1, -1, d).reshape(N, -1)
        dx = torch.where(live, grads[0], 0)
        _near(back[n], dx, u * dx.abs() + ((16 + d) * f + turn) * bound, "d" + n)
        if gn is not None:  # N * h terms in strands; every |term| <= |dy of its pair| |x^|
            terms = ((dy.view(N, h, d).norm(dim=-1) * math.sqrt(d))).sum()
            _near(dgain[n], grads[1], (f * (16 + math.sqrt(N * h)) + turn) * terms, "dgain_" + n)


@gpu
def test_qk_norm_rope_in_place_and_differences(pkg):
    """Results over their inputs are the same bits; a gradient agrees with central differences of the forward pass
    (step 2^-6: truncation 2^-12 of the third derivative, fp32 noise 2^-24 * 2^6)."""
    lib = pkg.library()
    case = (21, 3, 2, 32, 16, 0, 5, 0, 1)
    N, H, Hk, d = case[:4]
    for kind in KINDS:
        t, gain, pos = _norm_data(case, kind)
        shape = _norm_shape(pkg, case, kind)

        def forward(q, k, q_out, k_out):
            _ok(pkg, lib.nncu_qk_norm_rope_forward(C.byref(shape), _ptr(q), _ptr(k), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos), _ptr(q_out), _ptr(k_out), _stream()))
            return q_out, k_out

        apart = forward(t["q"], t["k"], torch.empty_like(t["q"]), torch.empty_like(t["k"]))
        q, k = t["q"].clone(), t["k"].clone()
        forward(q, k, q, k)
        assert torch.equal(q, apart[0]) and torch.equal(k, apart[1])
        need = C.c_size_t()
        _ok(pkg, lib.nncu_qk_norm_rope_workspace(C.byref(shape), C.byref(need)))
        room = torch.empty(need.value, dtype=torch.uint8, device="cuda")

        def backward(dq_out, dk_out, dq, dk):
            _ok(pkg, lib.nncu_qk_norm_rope_backward(C.byref(shape), _ptr(t["q"]), _ptr(t["k"]), _ptr(gain["q"]), _ptr(gain["k"]), _ptr(pos),
                                                    _ptr(dq_out), _ptr(dk_out), _ptr(dq), _ptr(dk), None, None, None, 0, _stream()))
            return dq, dk

        dq, dk = backward(t["dq_out"], t["dk_out"], torch.empty_like(t["q"]), torch.empty_like(t["k"]))
        over = t["dq_out"].clone(), t["dk_out"].clone()
        backward(*over, *over)
        assert torch.equal(over[0], dq) and torch.equal(over[1], dk)
        if kind == torch.float32:
            live = (pos >= 0)[:, None]
            g = torch.Generator(device="cuda").manual_seed(3)
            for i, (x, dx, dy) in enumerate(((t["q"], dq, t["dq_out"]), (t["k"], dk, t["dk_out"]))):
                way = torch.where(live, torch.randn(x.shape, generator=g, device="cuda"), 0)
                h = 2.0 ** -6
                ends = []
                for sign in (1, -1):
                    pair = [t["q"], t["k"]]
                    pair[i] = x + sign * h * way
                    ends.append(torch.where(live, forward(*pair, torch.empty_like(t["q"]), torch.empty_like(t["k"]))[i] * torch.where(live, dy, 0), 0).double().sum())
                slope = (ends[0] - ends[1]) / (2 * h)
                want = (dx.double() * way.double()).sum()
                assert abs(slope - want) < 2e-3 * (dx.double().norm() * way.double().norm()), (slope, want)


# ---------------------------------------------------------------- attention with a decaying state

def _form(a, b, c, s0, decay, length, scale_pair, scale_state, scale_in, reverse):
    """The chunk's form over whole streams, 64 bits: a, b [B][H][T][da], c [B][H][T][dc], s0 [B][H][da][dc] -> (o, state)"""
    B, H, T, _ = a.shape
    t = torch.arange(T, device=a.device)
    n = length[:, None]
    live = t < n                                             # [B][T]
    u = torch.where(live, (n - 1 - t) if reverse else t.expand(B, T), 0)
    rate = decay.double().log()[None, :, None]
    apart = (u[:, :, None] - u[:, None, :])[:, None]          # [B][1][T][T]
    both = (live[:, :, None] & live[:, None, :])[:, None] & (apart >= 0)
    w = torch.where(both, torch.exp(rate[..., None] * apart.clamp(min=0)), 0)
    a, b, c = (torch.where(live[:, None, :, None], x, 0) for x in (a, b, c))
    p = (a @ b.transpose(2, 3)) * w * scale_pair
    e1, e2 = (0, 1) if reverse else (1, 0)
    since = torch.where(live[:, None], torch.exp(rate * (u[:, None] + e1)), 0)[..., None]
    until = torch.where(live[:, None], torch.exp(rate * (n[:, None] - 1 - u[:, None] + e2)), 0)[..., None] * scale_in
    o = p @ c + since * (a @ s0) * scale_state
    return o, torch.exp(rate * n[:, None])[..., None] * s0 + (until * b).transpose(2, 3) @ c


LINEAR_CASES = [  # streams, heads, d_key, d_value, tokens, lengths, states
    (1, 1, 1, 1, 1, None, 1), (4, 4, 32, 32, 1, None, 1), (3, 2, 64, 128, 1, (1, 0, 1), 1), (2, 3, 24, 40, 2, None, 0), (2, 1, 128, 128, 8, (8, 5), 1),
    (2, 2, 16, 16, 9, (9, 0), 1), (1, 2, 64, 64, 63, None, 1), (3, 2, 64, 64, 64, None, 0), (2, 1, 64, 32, 65, (65, 64), 1), (1, 3, 32, 64, 128, (97,), 1),
    (2, 2, 128, 128, 130, (130, 1), 1), (1, 1, 128, 64, 200, None, 1), (2, 1, 8, 8, 77, (50, 77), 1), (1, 2, 96, 104, 150, (149,), 1),
    (1, 1, 5, 7, 100, None, 1), (1, 1, 64, 64, 1025, (1000,), 1), (2, 1, 128, 128, 700, (700, 333), 1), (1, 2, 32, 32, 513, None, 0),
    (5, 3, 40, 16, 300, (0, 300, 63, 64, 299), 1), (1, 1, 16, 128, 2048, None, 1), (150, 1, 64, 64, 100, None, 1),
    (2, 2, 40, 64, 333, (333, 100), 1), (13, 8, 64, 64, 50, (50, 0, 1, 49, 33, 50, 7, 50, 16, 17, 50, 2, 48), 1), (100, 1, 48, 56, 129, None, 0),
    (3, 1, 64, 40, 700, (700, 0, 257), 1)]


def _linear_data(case, kind, seed=5):
    B, H, dk, dv, T, length, states = case
    g = torch.Generator(device="cuda").manual_seed(seed + T + dk)

    def rows(d):
        return torch.randn(T * B, H * d, generator=g, device="cuda").to(kind)

    t = dict(q=rows(dk), k=rows(dk), v=rows(dv), dout=rows(dv))
    n = torch.tensor([T] * B if length is None else length, device="cuda")
    behind = (torch.arange(T, device="cuda")[:, None] >= n).reshape(T * B, 1)
    for x in t.values():
        x[behind.expand_as(x)] = float("nan")
    decay = torch.tensor([(0.9, 1.0, 0.999, 0.3, 1e-5)[(T + h) % 5] for h in range(H)])
    s0 = torch.randn(B, H, dk, dv, generator=g, device="cuda") if states else None
    ds = torch.randn(B, H, dk, dv, generator=g, device="cuda") if states else None
    return t, n, behind, decay, s0, ds, None if length is None else n.int()


class Linear:
    """The calls on one set of tensors, results in buffers that start as NaN"""

    def __init__(self, pkg, case, kind, t, decay, s0, ds, length, more=None):
        B, H, dk, dv, T = case[:5]
        self.pkg, self.t, self.decay, self.s0, self.ds, self.length = pkg, t, decay, s0, ds, length
        pitch = {n: x.stride(0) for n, x in t.items()}
        self.shape = pkg.abi.LinearAttnShape(n_streams=B, n_head=H, d_key=dk, d_value=dv, seg_len=T, ld_q=pitch["q"], ld_k=pitch["k"],
                                             ld_v=pitch["v"], ld_out=pitch["dout"], scale=dk ** -0.5, dtype_bf16=int(kind == torch.bfloat16))
        need = C.c_size_t()
        _ok(pkg, pkg.library().nncu_linear_attention_workspace(C.byref(self.shape), 1, C.byref(need)))
        self.need, self.room = need.value, torch.full((max(16, need.value),), 255, dtype=torch.uint8, device="cuda")
        like = lambda x: torch.full((x.shape[0], x.stride(0)), float("nan"), device="cuda", dtype=kind)[:, :x.shape[1]]  # noqa: E731
        self.out, self.dq, self.dk, self.dv = like(t["dout"]), like(t["q"]), like(t["k"]), like(t["v"])
        self.state, self.dstate = (torch.full((B, H, dk, dv), float("nan"), device="cuda") for _ in range(2))

    def forward(self, **over):
        a = {**self.t, "s0": self.s0, "out": self.out, "state": self.state, **over}
        _ok(self.pkg, self.pkg.library().nncu_linear_attention_forward(
            C.byref(self.shape), _ptr(a["q"]), _ptr(a["k"]), _ptr(a["v"]), self.decay.data_ptr(), _ptr(self.length), _ptr(a["s0"]), _ptr(a["out"]),
            _ptr(a["state"]), _ptr(self.room), self.need, _stream()))
        return a["out"], a["state"]

    def backward(self, **over):
        a = {**self.t, "s0": self.s0, "ds": self.ds, "dstate": self.dstate, **over}
        _ok(self.pkg, self.pkg.library().nncu_linear_attention_backward(
            C.byref(self.shape), _ptr(a["q"]), _ptr(a["k"]), _ptr(a["v"]), self.decay.data_ptr(), _ptr(self.length), _ptr(a["s0"]), _ptr(a["dout"]),
            _ptr(a["ds"]), _ptr(self.dq), _ptr(self.dk), _ptr(self.dv), _ptr(a["dstate"]), _ptr(self.room), self.need, _stream()))
        return self.dq, self.dk, self.dv, a["dstate"]


def _check_linear(pkg, case, kind, op, t, n, behind, decay, s0, ds):
    B, H, dk, dv, T = case[:5]
    scale = dk ** -0.5
    split = lambda x: torch.where(behind, 0, x).double().view(T, B, H, -1).permute(1, 2, 0, 3)  # noqa: E731
    join = lambda x: x.permute(2, 0, 1, 3).reshape(T * B, -1)  # noqa: E731
    q, k, v, do = (split(t[x]) for x in ("q", "k", "v", "dout"))
    zero = torch.zeros(B, H, dk, dv, device="cuda", dtype=torch.float64)
    s0, ds = (zero if x is None else x.double() for x in (s0, ds))
    d64 = decay.cuda().double()
    u, f = U[kind], 2.0 ** -23
    steps = max(dk, dv) + 64 + T / 16 + 40

    def both(*a):
        return _form(*a), _form(*(x.abs() if isinstance(x, torch.Tensor) and x.is_floating_point() else x for x in a))

    def rows_near(got, want, size, what):
        want, size = join(want), join(size)
        # one rounding of a weight to the operands' type: pair weights and states in bf16, nothing in fp32
        inner = U[kind] if kind == torch.bfloat16 else 0.0
        _near(got, want, u * want.abs() + (1.01 * inner + steps * f) * size + 1e-30, what)

    (out, state), (out_, state_) = both(q, k, v, s0, d64, n, scale, scale, 1.0, False)
    got = op.forward()
    rows_near(got[0], out, out_, "out")
    _near(got[1], state, (T + 64) * f * state_ + 1e-30, "state")
    t_ = lambda x: x.transpose(2, 3)  # noqa: E731
    dq, dk_, dv_, dstate = op.backward()
    (want, _), (size, _) = both(do, v, k, t_(s0), d64, n, scale, scale, 1.0, False)
    rows_near(dq, want, size, "dq")
    (want, _), (size, _) = both(v, do, q, t_(ds), d64, n, scale, 1.0, scale, True)
    rows_near(dk_, want, size, "dk")
    (want, last), (size, last_) = both(k, q, do, ds, d64, n, scale, 1.0, scale, True)
    rows_near(dv_, want, size, "dv")
    _near(dstate, last, (T + 64) * f * last_ + 1e-30, "dstate")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", LINEAR_CASES)
def test_linear_attention_against_64_bits(pkg, case, kind):
    """One token to long texts, head sizes that fill no tile, streams that end inside a chunk or have no token, decays
    from none to none left after a token, padding that holds NaN."""
    t, n, behind, decay, s0, ds, length = _linear_data(case, kind)
    _check_linear(pkg, case, kind, Linear(pkg, case, kind, t, decay, s0, ds, length), t, n, behind, decay, s0, ds)


@gpu
@pytest.mark.parametrize("case", [
    (1, 2, 128, 128, 200, None, 1), (2, 1, 4, 128, 65, (65, 32), 1), (1, 2, 128, 4, 97, None, 0), (3, 2, 36, 100, 130, (130, 0, 31), 1),
    (40, 4, 12, 20, 33, None, 1), (1, 1, 112, 116, 1000, (993,), 1), (2, 4, 68, 60, 300, (300, 129), 1), (60, 4, 64, 64, 40, None, 1)])
def test_linear_attention_fp32_sizes(pkg, case):
    """fp32 head sizes about the tiles of its products.  A product of two values in two parts of 11 bits is off by 2^-22 of it
    for the part left out and 2^-23 for each rest: less than the steps that the tolerance counts"""
    t, n, behind, decay, s0, ds, length = _linear_data(case, torch.float32, seed=6)
    _check_linear(pkg, case, torch.float32, Linear(pkg, case, torch.float32, t, decay, s0, ds, length), t, n, behind, decay, s0, ds)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 70, 600])
@pytest.mark.parametrize("shift", [0, 1])
def test_linear_attention_in_one_buffer(pkg, kind, T, shift):
    """q, k, v as column groups of one buffer, which begins at and between 16-byte boundaries"""
    case = (2, 3, 32, 48, T, None, 1)
    B, H, dk, dv = case[:4]
    t, n, behind, decay, s0, ds, length = _linear_data(case, kind)
    wide = H * (2 * dk + dv) + 8 + shift
    buf = torch.full((T * B * wide + 8,), float("nan"), device="cuda", dtype=kind)[shift:shift + T * B * wide].view(T * B, wide)
    at = 0
    for x in ("q", "k", "v"):
        w = t[x].shape[1]
        buf[:, at:at + w] = t[x]
        t[x] = buf[:, at:at + w]
        at += w
    before = buf.clone()
    _check_linear(pkg, case, kind, Linear(pkg, case, kind, t, decay, s0, ds, length), t, n, behind, decay, s0, ds)
    assert torch.equal(torch.nan_to_num(buf.float()), torch.nan_to_num(before.float()))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 5, 64, 1500])
def test_linear_attention_state_in_place(pkg, kind, T):
    """state_out over state_in, dstate_in over dstate_out: the bits of separate buffers; lengths past the ends are taken
    into the segment; the same call again gives the same bits"""
    case = (3, 2, 64, 64, T, None, 1)
    t, n, behind, decay, s0, ds, _ = _linear_data(case, kind)
    length = torch.tensor([T + 5, -2, T], device="cuda").int()
    op = Linear(pkg, case, kind, t, decay, s0, ds, length)
    out, state = (x.clone() for x in op.forward())
    assert torch.equal(state[1], s0[1]) and bool((out.view(T, 3, -1)[:, 1] == 0).all())
    over = s0.clone()
    op.forward(s0=over, state=over)
    assert torch.equal(over, state) and torch.equal(op.out, out)
    grads = [x.clone() for x in op.backward()]
    over = ds.clone()
    again = op.backward(ds=over, dstate=over)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@gpu
def test_linear_attention_segments_carry_the_state(pkg):
    """A text in pieces of 1, 7, 64 and 130 tokens with the state carried on, against the text in one call: fp32, the same
    sums in another order (2^-24 a step, 400 steps)"""
    pieces = (1, 7, 64, 130)
    T, case = sum(pieces), (2, 2, 32, 32, sum(pieces), None, 1)
    t, n, behind, decay, s0, ds, _ = _linear_data(case, torch.float32)
    out, state = Linear(pkg, case, torch.float32, t, decay, s0, ds, None).forward()
    carried, at, rows = s0.clone(), 0, []
    for m in pieces:
        part = {x: y[at * 2:(at + m) * 2] for x, y in t.items()}
        op = Linear(pkg, (2, 2, 32, 32, m), torch.float32, part, decay, carried, ds, None)
        rows.append(op.forward(state=carried)[0].clone())
        at += m
    size = out.abs().max().item()
    assert (torch.cat(rows) - out).abs().max().item() < 400 * 2.0 ** -24 * 8 * size
    assert (carried - state).abs().max().item() < 400 * 2.0 ** -24 * 8 * state.abs().max().item()


@gpu
def test_linear_attention_gradients_against_differences(pkg):
    """The result is linear in q, in k, in v and in the state: a whole step along a way changes sum(out dout) +
    sum(state dstate) by the gradient's share of it, up to fp32 sums"""
    case = (2, 2, 32, 48, 90, (90, 33), 1)
    t, n, behind, decay, s0, ds, length = _linear_data(case, torch.float32)
    op = Linear(pkg, case, torch.float32, t, decay, s0, ds, length)
    grads = dict(zip(("q", "k", "v", "s0"), (x.clone().double() for x in op.backward())))
    do = torch.where(behind, 0, t["dout"]).double()

    def value(**over):
        out, state = op.forward(**over)
        return (out.double() * do).sum() + (state.double() * ds.double()).sum()

    g = torch.Generator(device="cuda").manual_seed(9)
    base = value()
    for name, x in (("q", t["q"]), ("k", t["k"]), ("v", t["v"]), ("s0", s0)):
        way = torch.randn(x.shape, generator=g, device="cuda")
        want = (torch.where(behind, 0, way).double() * grads[name]).sum() if name != "s0" else (way.double() * grads[name]).sum()
        assert abs(value(**{name: x + way}) - base - want) < 1e-4 * grads[name].norm() * way.double().norm(), name


# ---------------------------------------------------------------- the loss against a teacher's top logits

def _distill_ref(z, ids, top, targets, weight, tau, share):
    """(losses, gradient) in 64 bits"""
    N, V = z.shape
    z = z.double().clone()
    empty = (z == -math.inf).all(1) | (weight == 0)
    z[empty] = 0
    z.requires_grad_()
    there = (ids >= 0) & (ids < V)
    known = (targets >= 0) & (targets < V)
    log_hard, log_soft = torch.log_softmax(z, 1), torch.log_softmax(z / tau, 1)
    log_q = torch.log_softmax(torch.where(there, top.double() / tau, -1e30), 1) if ids.shape[1] else top.double()
    q = torch.where(there, log_q.exp(), 0)
    kl = torch.where(q > 0, q * (log_q - log_soft.gather(1, torch.where(there, ids, 0).long())), 0).sum(1)
    miss = torch.where(known, -log_hard.gather(1, torch.where(known, targets, 0).long()[:, None])[:, 0], 0)
    loss = torch.where(empty, 0, weight.double() * ((1 - share) * miss + share * tau ** 2 * kl))
    grad, = torch.autograd.grad(loss.sum(), z) if loss.requires_grad else (torch.zeros_like(z),)
    return loss.detach(), torch.where(empty[:, None], 0, grad)


def _distill_data(N, V, K, kind, seed=2):
    g = torch.Generator(device="cuda").manual_seed(seed + N + V)
    z = 3 * torch.randn(N, V, generator=g, device="cuda")
    ids = torch.randint(0, V, (N, K), generator=g, device="cuda").int()  # some symbols more than once
    top = 2 * torch.randn(N, K, generator=g, device="cuda")
    targets = torch.randint(0, V, (N,), generator=g, device="cuda").int()
    if K:
        targets[::2] = ids[::2, 0]
    weight = torch.rand(N, generator=g, device="cuda") + 0.1
    return z.to(kind), ids, top, targets, weight


def _distill_calls(pkg, z, ids, top, targets, weight, tau, share, grad_kind, ld=0):
    """Losses and gradient of the fused call, gradient of the pair of calls"""
    lib = pkg.library()
    N, V = z.shape
    K = ids.shape[1]
    shape = pkg.abi.DistillShape(n_rows=N, n_symbols=V, n_top=K, ld_logits=z.stride(0), ld_dlogits=ld, temperature=tau, teacher_share=share,
                                 logits_bf16=int(z.dtype == torch.bfloat16), grad_bf16=int(grad_kind == torch.bfloat16))
    new = lambda: torch.full((N, ld or V), 7.0, device="cuda", dtype=grad_kind)  # noqa: E731
    loss, loss2, lse = (torch.full((N * k,), float("nan"), device="cuda") for k in (1, 1, 2))
    dz, dz2 = new(), new()
    args = (_ptr(z), _ptr(ids), _ptr(top), _ptr(targets), _ptr(weight))
    _ok(pkg, lib.nncu_distill_gradient(C.byref(shape), *args, _ptr(loss), _ptr(dz), _stream()))
    _ok(pkg, lib.nncu_distill_forward(C.byref(shape), *args, _ptr(loss2), _ptr(lse), _stream()))
    _ok(pkg, lib.nncu_distill_backward(C.byref(shape), *args, _ptr(lse), _ptr(dz2), _stream()))
    if ld:
        assert bool((dz[:, V:] == 7).all()) and bool((dz2[:, V:] == 7).all())
    assert bool(((loss == loss2) | ((loss - loss2).abs() < 1e-5 * (1 + loss.abs()))).all())
    return loss, dz[:, :V], dz2[:, :V]


def _distill_near(loss, dzs, want, grad, weight, tau, share, kind, V):
    # a loss is a difference of logs of sums of V terms: 2^-24 for each of about thirty steps of the tree, of sizes to tau^2 * 30
    _near(loss, want, 2.0 ** -24 * 60 * (want.abs() + weight.double() * (30 + 30 * tau * tau)), "loss")
    # a probability: fp32 exponentials of differences to 40 (2^-24 * 64 of it); their weighted sum, rounded once
    size = weight.double()[:, None] * (1 + share * tau)
    for dz in dzs:
        _near(dz, grad, U[kind] * grad.abs() + 2.0 ** -24 * 128 * size, "dlogits")


@gpu
@pytest.mark.parametrize("N,V,K,kind,grad_kind,tau,share", [
    (1, 1, 0, torch.float32, torch.float32, 1.0, 0.0), (7, 2, 2, torch.float32, torch.float32, 1.0, 0.5), (128, 256, 16, torch.float32, torch.bfloat16, 2.0, 0.7),
    (33, 257, 100, torch.float32, torch.float32, 0.5, 1.0), (20, 255, 30, torch.bfloat16, torch.bfloat16, 1.0, 0.3), (9, 2048, 64, torch.bfloat16, torch.float32, 3.0, 0.5),
    (9, 2049, 64, torch.float32, torch.float32, 1.0, 0.5), (5, 4100, 50, torch.bfloat16, torch.bfloat16, 2.0, 0.9), (3, 9208, 50, torch.bfloat16, torch.bfloat16, 2.0, 0.9),
    (4, 16384, 128, torch.float32, torch.bfloat16, 2.0, 0.7), (2, 16385, 40, torch.float32, torch.float32, 1.0, 0.5), (2, 50000, 1024, torch.float32, torch.bfloat16, 4.0, 0.5),
    (3, 40001, 7, torch.bfloat16, torch.bfloat16, 1.0, 1.0), (6, 6609, 21, torch.bfloat16, torch.float32, 2.0, 0.4)])
def test_distillation_against_64_bits(pkg, N, V, K, kind, grad_kind, tau, share):
    z, ids, top, targets, weight = _distill_data(N, V, K, kind)
    got = _distill_calls(pkg, z, ids, top, targets, weight, tau, share, grad_kind)
    want, grad = _distill_ref(z, ids, top, targets, weight, tau, share)
    _distill_near(got[0], got[1:], want, grad, weight, tau, share, grad_kind, V)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [64, 300, 4096, 20000])
def test_distillation_masks(pkg, kind, V):
    """Symbols masked out, rows of nothing but them, teachers that sent fewer entries or none, -inf among their logits, no
    target, weight 0 over NaN logits, rows with a pitch"""
    N, K = 12, 20
    z, ids, top, targets, weight = _distill_data(N, V, K, kind, seed=4)
    buf = torch.full((N, V + 12), float("nan"), device="cuda", dtype=kind)
    buf[:, :V] = z
    z = buf[:, :V]
    z[0] = -math.inf                                     # nothing left
    z[1, V // 2:] = -math.inf                             # half of the alphabet
    ids[1], targets[1] = ids[1] % (V // 2), targets[1] % (V // 2)
    z[2] = -math.inf
    z[2, 5] = 1.0                                        # one symbol left
    ids[2], targets[2] = 5, 5
    ids[3] = -1                                          # no teacher
    ids[4, K // 2:] = V + 3                               # fewer entries
    top[4, K // 2:] = float("nan")
    top[5, 3:] = -math.inf                                # entries that cannot come
    top[6] = -math.inf                                    # none that can
    targets[7] = -1
    targets[8] = V
    ids[9], targets[9] = -1, -1                            # neither
    weight[10], z[10] = 0, float("nan")
    ids[11, :] = ids[11, 0]                               # one symbol, K times
    want, grad = _distill_ref(z, torch.where((top == -math.inf) & (top == -math.inf).all(1, keepdim=True), -1, ids), torch.where(ids < V, top, 0), targets, weight, 2.0, 0.6)
    got = _distill_calls(pkg, z, ids, top, targets, weight, 2.0, 0.6, kind, ld=V + 4)
    for x in got:
        assert bool((x[0] == 0).all()) and bool((x[9] == 0).all()) and bool((x[10] == 0).all())
    for x in got[1:]:
        assert bool((x[1, V // 2:] == 0).all())
    _distill_near(got[0], got[1:], want, grad, weight, 2.0, 0.6, kind, V)


@gpu
@pytest.mark.parametrize("N,V,K,kind,grad_kind,tau,share", [
    (5000, 300, 20, torch.bfloat16, torch.bfloat16, 2.0, 0.7), (5000, 256, 200, torch.float32, torch.float32, 1.0, 0.5), (1400, 4096, 50, torch.float32, torch.bfloat16, 3.0, 0.7),
    (1000, 16384, 64, torch.bfloat16, torch.float32, 2.0, 0.4), (500, 16385, 300, torch.float32, torch.bfloat16, 2.0, 1.0)])
def test_distillation_of_more_rows_than_places(pkg, N, V, K, kind, grad_kind, tau, share):
    """Rows that follow one another on an SM: some of them masked out, without a teacher or of weight 0, with symbols that
    several entries name"""
    z, ids, top, targets, weight = _distill_data(N, V, K, kind, seed=12)
    ids[1::3, 1::2] = ids[1::3, :1]
    ids[5::13] = -1
    targets[4::9] = V
    z[3::11] = -math.inf
    weight[2::7] = 0.0
    got = _distill_calls(pkg, z, ids, top, targets, weight, tau, share, grad_kind)
    want, grad = _distill_ref(z, ids, top, targets, weight, tau, share)
    _distill_near(got[0], got[1:], want, grad, weight, tau, share, grad_kind, V)


@gpu
def test_distillation_without_targets_or_weights(pkg):
    z, ids, top, _, _ = _distill_data(6, 100, 10, torch.float32)
    got = _distill_calls(pkg, z, ids, top, None, None, 1.0, 1.0, torch.float32)
    one = torch.ones(6, device="cuda")
    want, grad = _distill_ref(z, ids, top, torch.full((6,), -1, device="cuda"), one, 1.0, 1.0)
    _distill_near(got[0], got[1:], want, grad, one, 1.0, 1.0, torch.float32, 100)
    # a logit that the teacher wants and the mask forbids: the loss is infinite, the gradient is not
    z[0, ids[0, 0].long()] = -math.inf
    loss, dz, dz2 = _distill_calls(pkg, z, ids, top, None, None, 1.0, 1.0, torch.float32)
    assert loss[0] == math.inf and bool(torch.isfinite(loss[1:]).all()) and bool(torch.isfinite(dz).all()) and bool(torch.isfinite(dz2).all())


@gpu
def test_distillation_gradient_against_differences(pkg):
    """Central differences of the losses (step 2^-5: truncation 2^-10 / 6 of third derivatives below 1)"""
    z, ids, top, targets, weight = _distill_data(8, 64, 12, torch.float32)
    _, dz, _ = _distill_calls(pkg, z, ids, top, targets, weight, 2.0, 0.5, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(1)
    way, h = torch.randn(z.shape, generator=g, device="cuda"), 2.0 ** -5
    up, down = (_distill_calls(pkg, z + s * h * way, ids, top, targets, weight, 2.0, 0.5, torch.float32)[0].double() for s in (1, -1))
    slope, want = (up - down) / (2 * h), (dz.double() * way.double()).sum(1)
    assert (slope - want).abs().max() < 5e-3 * (1 + want.abs().max())


# ---------------------------------------------------------------- together, and as programs call them

def _student(pkg, seed=0):
    """One training step of a student: norm with rotation, attention, output matrix, loss, and back, on the library's calls"""
    lib = pkg.library()
    B, H, d, T, V, K = 3, 2, 32, 40, 120, 8
    D, N = H * d, T * B
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s, scale=1.0: scale * torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kind = torch.bfloat16
    q, k, v = (rnd(N, D).to(kind) for _ in range(3))
    gain = 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d)
    w = rnd(V, D, scale=0.2).to(kind)
    pos = torch.arange(T, device="cuda").repeat_interleave(B).int()
    decay = torch.tensor([0.9, 0.99])
    ids, top = torch.randint(0, V, (N, K), generator=g, device="cuda").int(), rnd(N, K)
    targets = torch.randint(0, V, (N,), generator=g, device="cuda").int()
    ns = pkg.abi.QkNormShape(n_rows=N, n_head=H, n_head_k=H, d_key=d, d_rot=d, eps=1e-6, rope_base=1e4, dtype_bf16=1)
    ls = pkg.abi.LinearAttnShape(n_streams=B, n_head=H, d_key=d, d_value=d, seg_len=T, scale=d ** -0.5, dtype_bf16=1)
    ds = pkg.abi.DistillShape(n_rows=N, n_symbols=V, n_top=K, temperature=2.0, teacher_share=0.5, logits_bf16=0, grad_bf16=1)
    need, need2 = C.c_size_t(), C.c_size_t()
    _ok(pkg, lib.nncu_qk_norm_rope_workspace(C.byref(ns), C.byref(need)))
    _ok(pkg, lib.nncu_linear_attention_workspace(C.byref(ls), 1, C.byref(need2)))
    room = torch.empty(max(need.value, need2.value, 16), dtype=torch.uint8, device="cuda")
    e = lambda *s, t=kind: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
    b = dict(qn=e(N, D), kn=e(N, D), o=e(N, D), state=e(B, H, d, d, t=torch.float32), z=e(N, V, t=torch.float32), loss=e(N, t=torch.float32),
             dz=e(N, V), do=e(N, D), dw=e(V, D, t=torch.float32), dqn=e(N, D), dkn=e(N, D), dv=e(N, D), dq=e(N, D), dk=e(N, D),
             gq=e(d, t=torch.float32), gk=e(d, t=torch.float32))

    def norm_attention(st):
        _ok(pkg, lib.nncu_qk_norm_rope_forward(C.byref(ns), _ptr(q), _ptr(k), _ptr(gain[0]), _ptr(gain[1]), _ptr(pos), _ptr(b["qn"]), _ptr(b["kn"]), st))
        _ok(pkg, lib.nncu_linear_attention_forward(C.byref(ls), _ptr(b["qn"]), _ptr(b["kn"]), _ptr(v), decay.data_ptr(), None, None, _ptr(b["o"]),
                                                   _ptr(b["state"]), _ptr(room), need2.value, st))

    def head(st):
        _ok(pkg, lib.nncu_gemm_bf16(pkg.abi.GEMM_AUTO, 0, N, V, D, _ptr(b["o"]), D, _ptr(w), D, _ptr(b["z"]), V, 1, st))

    def loss(st):
        _ok(pkg, lib.nncu_distill_gradient(C.byref(ds), _ptr(b["z"]), _ptr(ids), _ptr(top), _ptr(targets), None, _ptr(b["loss"]), _ptr(b["dz"]), st))

    def head_back(st):
        _ok(pkg, lib.nncu_gemm_bf16(pkg.abi.GEMM_AUTO, 1, N, D, V, _ptr(b["dz"]), V, _ptr(w), D, _ptr(b["do"]), D, 0, st))
        _ok(pkg, lib.nncu_gemm_bf16(pkg.abi.GEMM_AUTO, 2, V, D, N, _ptr(b["dz"]), V, _ptr(b["o"]), D, _ptr(b["dw"]), D, 1, st))

    def back(st):
        _ok(pkg, lib.nncu_linear_attention_backward(C.byref(ls), _ptr(b["qn"]), _ptr(b["kn"]), _ptr(v), decay.data_ptr(), None, None, _ptr(b["do"]),
                                                    None, _ptr(b["dqn"]), _ptr(b["dkn"]), _ptr(b["dv"]), None, _ptr(room), need2.value, st))
        _ok(pkg, lib.nncu_qk_norm_rope_backward(C.byref(ns), _ptr(q), _ptr(k), _ptr(gain[0]), _ptr(gain[1]), _ptr(pos), _ptr(b["dqn"]), _ptr(b["dkn"]),
                                                _ptr(b["dq"]), _ptr(b["dk"]), _ptr(b["gq"]), _ptr(b["gk"]), _ptr(room), need.value, st))

    keep = (q, k, v, gain, w, pos, decay, ids, top, targets, room, ns, ls, ds)
    return b, (norm_attention, head, loss, head_back, back), keep, (B, H, d, T, V)


@gpu
def test_a_student_step_and_its_gradients(pkg):
    """The operators together, against 64-bit autograd of the whole step.  Every stage rounds to bf16 (2^-8): the bound is
    eight such roundings of the gradient's norm."""
    b, stages, keep, (B, H, d, T, V) = _student(pkg)
    for f in stages:
        f(_stream())
    q, k, v, gain, w, pos, decay, ids, top, targets = keep[:10]
    leaves = [x.double().requires_grad_() for x in (q, k, v, gain[0], gain[1], w)]
    q6, k6, v6, gq, gk, w6 = leaves
    qn, kn = (_norm_ref(x, gx, pos, d, d, 0, 1e-6, 1e4) for x, gx in ((q6, gq), (k6, gk)))
    split = lambda x: x.view(T, B, H, d).permute(1, 2, 0, 3)  # noqa: E731
    zero = torch.zeros(B, H, d, d, device="cuda", dtype=torch.float64)
    o, _ = _form(split(qn), split(kn), split(v6), zero, decay.cuda().double(), torch.full((B,), T, device="cuda"), d ** -0.5, d ** -0.5, 1.0, False)
    z = o.permute(2, 0, 1, 3).reshape(T * B, -1) @ w6.T
    log_hard, log_soft = torch.log_softmax(z, 1), torch.log_softmax(z / 2, 1)
    log_q = torch.log_softmax(top.double() / 2, 1)
    loss = 0.5 * -log_hard.gather(1, targets.long()[:, None])[:, 0] + 0.5 * 4 * (log_q.exp() * (log_q - log_soft.gather(1, ids.long()))).sum(1)
    grads = torch.autograd.grad(loss.sum(), leaves)
    assert ((b["loss"].double() - loss).norm() / loss.norm()).item() < 8 * 2.0 ** -8
    for name, want in zip(("dq", "dk", "dv", "gq", "gk", "dw"), grads):
        assert ((b[name].double() - want).norm() / want.norm()).item() < 8 * 2.0 ** -8, name


@gpu
def test_captured_and_replayed_on_another_stream(pkg):
    """Stages of a step captured on a stream of their own while an eager step of the same tensors has run, replayed twice:
    the bits of the eager step.  (The products between them wait for the GPU, so they stay outside the graphs.)"""
    b, stages, keep, _ = _student(pkg, 3)
    for f in stages:
        f(_stream())
    torch.cuda.synchronize()
    eager = {n: x.clone() for n, x in b.items()}
    side = torch.cuda.Stream()
    graphs = {}
    for i in (0, 2, 4):
        graphs[i] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[i], stream=side):
            stages[i](_stream())
    for _ in range(2):
        for x in b.values():
            x.fill_(float("nan"))
        for i, f in enumerate(stages):
            graphs[i].replay() if i in graphs else f(_stream())
        torch.cuda.synchronize()
        for n, x in b.items():
            assert torch.equal(x, eager[n]), n


@gpu
def test_two_streams_at_once(pkg):
    """Two steps with workspaces of their own side by side give the bits of one after the other"""
    one, two = _student(pkg, 5), _student(pkg, 6)
    want = []
    for b, stages, _, _ in (one, two):
        for f in stages:
            f(_stream())
        torch.cuda.synchronize()
        want.append({n: x.clone() for n, x in b.items()})
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for i in (0, 2, 4):
            for (b, stages, _, _), st in zip((one, two), streams):
                stages[i](st.cuda_stream)
    torch.cuda.synchronize()
    for (b, *_), w in zip((one, two), want):
        for n, x in b.items():
            assert torch.equal(x, w[n]), n


# ---------------------------------------------------------------- the model's own path

@gpu
@pytest.mark.parametrize("bf16,V", [(0, 256), (0, 1024), (1, 300)])
def test_model_learns_from_a_teacher(pkg, bf16, V):
    """The gradient is linear in what a row is to predict: a teacher with the same q in every row gives the weighted sum of the
    gradients of its symbols as targets, (1 - share) of the target's beside it; the loss is the weighted sum of theirs
    less share sum q ln q a row.  fp32: sums in another order (2^-24 times some thousand terms); bf16: a rounding of every
    operand, 2^-8, in each of two layers."""
    np = pytest.importorskip("numpy")
    kw = dict(n_layer=2, d_model=64, n_head=2, d_key=32, d_inner=128, d_pos=24, mem_len=16, seg_len=16, n_streams=4, n_symbols=V,
              use_bf16=bf16, init_range=0.2)
    T, B, K, share = 16, 4, 3, 0.6
    rng = np.random.default_rng(V)
    m = pkg.TrfModel(pkg.abi.make_params(**kw))
    m.reset()
    m._ck(m.lib.nncu_own_stream(m.h))
    logits = np.array([0.3, -1.0, 0.8], np.float32)
    q = np.exp(logits.astype(np.float64)); q /= q.sum()
    tol = 4e-2 if bf16 else 2e-4
    for step in range(4):  # eager, captured, replayed, both memory twins
        ids_in = rng.integers(0, V, (T, B)).astype(np.int32)
        tg = rng.integers(0, V, (T, B)).astype(np.int32)
        top = np.stack([rng.permutation(V)[:K] for _ in range(T * B)]).reshape(T, B, K).astype(np.int32)
        top[0, 0] = tg[0, 0]            # the target three times
        top[1, 1, 1] = top[1, 1, 0]     # a symbol twice
        rows = np.broadcast_to(logits, (T, B, K)).copy()
        m.eval(-1, ids_in, read=False)
        loss_t = m.eval_gradient(tg)
        want = {n: (1 - share) * m.get_grad(n).astype(np.float64) for n in m.info}
        loss = (1 - share) * loss_t
        for k in range(K):
            loss += share * q[k] * m.eval_gradient(np.ascontiguousarray(top[:, :, k]))
            for n in want:
                want[n] += share * q[k] * m.get_grad(n)
        loss -= share * (q * np.log(q)).sum() * T * B
        got = m.eval_gradient_distill(tg, top, rows, share)
        assert abs(got - loss) < tol * abs(loss), (got, loss)
        for n in want:
            scale = max(np.abs(want[n]).max(), 1e-9)
            assert np.abs(m.get_grad(n) - want[n]).max() < tol * scale, n
        # entries outside the alphabet: no teacher; and the plain loss behind a teacher's is what it was before
        plain = {n: m.get_grad(n) for n in m.info} if m.eval_gradient(tg) == loss_t else None
        assert plain is not None
        assert m.eval_gradient_distill(tg, np.full((T, B, K), -1, np.int32), rows, share) == loss_t
        for n in plain:
            assert np.array_equal(m.get_grad(n), plain[n]), n
        m.update()
    with pytest.raises(Exception):
        m.eval_gradient_distill(tg, top, rows, 1.5)
    m.close()


def test_model_distillation_refuses_bad_arguments(pkg):
    import ctypes
    lib = pkg.library()
    one, loss = 4096, ctypes.c_float()
    assert lib.nncu_eval_gradient_distill(None, one, 1, one, one, 0.5, ctypes.byref(loss)) == pkg.abi.ERR_INVALID


# ---------------------------------------------------------------- offsets beyond 32 bits

@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_rows_far_apart(pkg, kind):
    """Row pitches that put rows more than 2^32 bytes from the first: the bits of rows that lie close together"""
    B, T, d = 2, 1100, 64
    N, pitch = B * T, 1 << (20 if kind == torch.bfloat16 else 19)
    buf = torch.empty(N * pitch, device="cuda", dtype=kind).view(N, pitch)
    assert N * pitch * buf.element_size() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(4)
    near, far = {}, {}
    for i, x in enumerate(("q", "k", "v", "dout")):
        near[x] = torch.randn(N, d, generator=g, device="cuda").to(kind)
        far[x] = buf[:, 4096 * i:4096 * i + d]
        far[x].copy_(near[x])
    decay, s0 = torch.tensor([0.97]), torch.randn(B, 1, d, d, generator=g, device="cuda")
    results = []
    for t in (near, far):
        op = Linear(pkg, (B, 1, d, d, T), kind, t, decay, s0, s0.clone(), None)
        op.out = torch.empty(N, d, device="cuda", dtype=kind) if t is near else buf[:, 32768:32768 + d]
        if t is far:
            op.dq, op.dk, op.dv = (buf[:, 40000 + 1000 * i:40000 + 1000 * i + d] for i in range(3))
        results.append([x.clone() for x in (*op.forward(), *op.backward())])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # norms of rows that far apart, and logits
    pos = torch.arange(N, device="cuda").int()
    outs = []
    for t in (near, far):
        p = t["q"].stride(0)
        s = pkg.abi.QkNormShape(n_rows=N, n_head=1, n_head_k=1, d_key=d, d_rot=d, ld_q=p, ld_k=p, ld_q_out=p, ld_k_out=p, eps=1e-6, rope_base=1e4,
                                dtype_bf16=int(kind == torch.bfloat16))
        q, k = (torch.empty(N, d, device="cuda", dtype=kind) for _ in range(2)) if t is near else (buf[:, 50000 + 1000 * i:50000 + 1000 * i + d] for i in range(2))
        _ok(pkg, pkg.library().nncu_qk_norm_rope_forward(C.byref(s), _ptr(t["q"]), _ptr(t["k"]), None, None, _ptr(pos), _ptr(q), _ptr(k), _stream()))
        outs.append((q.clone(), k.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    z, ids, top, targets, weight = _distill_data(N, 2000, 20, kind)
    far_z = buf[:, 100000:102000]
    far_z.copy_(z)
    one, two = (_distill_calls(pkg, x, ids, top, targets, weight, 2.0, 0.5, kind) for x in (z, far_z))
    assert all(torch.equal(a, b) for a, b in zip(one, two))
