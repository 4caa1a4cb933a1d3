"""The operators of a student model, as cases that can be timed and compared.

  norm      queries and keys normed for each head and rotated by their positions in the same pass
  linear    attention with a state that decays at each head's own rate: one token, a segment, a long text, with
            the state carried from call to call; with train, the backward pass too
  distill   the loss of a student against a teacher's top logits mixed with the coded symbol's own, and its gradient

Rows are (time, stream) positions, row = time * n_streams + stream, as everywhere in the library.  Streams of a
padded batch end early: their rows behind the end hold whatever memory held (NaN here), and results there are zeros.
"""
import ctypes as C
import importlib.util
import math
import os
import sys

import torch

own = False


def _package():
    """The package of the repository in the working folder (its folder's name is not an identifier)."""
    name = "nncp_metal_b200"
    if name not in sys.modules:
        folder = os.path.abspath("nncp-metal_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules[name] = module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    return sys.modules[name]


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one token of the smallest models (fp32 heads of 32): a call is its latency
        dict(name="linear token config0", kind="linear", n_streams=4, n_head=4, d_key=32, d_value=32, seg_len=1, bf16=0,
             ragged=0, state=1, train=0),
        # one token of many streams: every stream's state through the chip
        dict(name="linear token config4", kind="linear", n_streams=128, n_head=8, d_key=64, d_value=64, seg_len=1, bf16=1,
             ragged=0, state=1, train=0),
        # a segment of the text model, its state carried from the segment before to the one behind
        dict(name="linear segment config2", kind="linear", n_streams=32, n_head=8, d_key=64, d_value=64, seg_len=64, bf16=1,
             ragged=0, state=1, train=0),
        # two long texts read from their beginnings by a model of wide heads
        dict(name="linear long texts", kind="linear", n_streams=2, n_head=8, d_key=128, d_value=128, seg_len=4096, bf16=1,
             ragged=0, state=1, train=0),
        # a training step of tokenised text: lengths that fill no tile, streams that end early
        dict(name="linear train words", kind="linear", n_streams=13, n_head=8, d_key=64, d_value=64, seg_len=50, bf16=1,
             ragged=1, state=1, train=1),
        # a training step over long segments of the deep model's heads
        dict(name="linear train long", kind="linear", n_streams=8, n_head=16, d_key=64, d_value=64, seg_len=2048, bf16=1,
             ragged=0, state=0, train=1),
        # a step of the default level's fp32 model
        dict(name="norm train level6", kind="norm", n_rows=512, n_head=8, n_head_k=8, d_key=32, d_rot=32, adjacent=0, bf16=0,
             far=0, ragged=0, train=1),
        # a segment of tokenised text far into a large file, some rows padding, keys of fewer heads
        dict(name="norm words", kind="norm", n_rows=650, n_head=8, n_head_k=2, d_key=64, d_rot=64, adjacent=1, bf16=1, far=1,
             ragged=1, train=0),
        # a training step of long segments of the large model
        dict(name="norm train config3", kind="norm", n_rows=16384, n_head=16, n_head_k=16, d_key=64, d_rot=32, adjacent=0,
             bf16=1, far=0, ragged=0, train=1),
        # bytes, the smallest model: loss and gradient of one segment
        dict(name="distill config0", kind="distill", n_rows=128, n_symbols=256, n_top=16, temperature=1.0, teacher=0.5,
             bf16=0, grad_bf16=0, ragged=0, apart=0),
        # tokenised text: an alphabet that is no power of two with symbols masked out, padded rows, loss and gradient apart
        dict(name="distill words", kind="distill", n_rows=650, n_symbols=9208, n_top=50, temperature=2.0, teacher=0.9,
             bf16=1, grad_bf16=1, ragged=1, apart=1),
        # the text model that the headline figure is quoted on: fp32 logits, bf16 gradient
        dict(name="distill config2", kind="distill", n_rows=2048, n_symbols=16384, n_top=64, temperature=2.0, teacher=0.7,
             bf16=0, grad_bf16=1, ragged=0, apart=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _drawn(rng)
        # no more than the largest listed case has: bytes, and for the plain form every pair of a stream's rows
        pairs = c["n_streams"] * c["n_head"] * c["seg_len"] ** 2 * (c["d_key"] + c["d_value"]) if c["kind"] == "linear" else 0
        if work(c)["bytes"] <= 2.7e8 and pairs <= 6.8e10:
            return c


def _drawn(rng):
    kind = rng.choice(("linear",) * 5 + ("norm",) * 3 + ("distill",) * 3)
    if kind == "linear":
        bf16 = int(rng.random() < 0.8)
        d_key = rng.choice((16, 32, 64, 64, 128, 128, 8 * rng.randint(1, 16)))
        d_value = d_key if rng.random() < 0.7 else rng.choice((32, 64, 128, 8 * rng.randint(1, 16)))
        c = dict(kind=kind, n_head=_log_int(rng, 1, 16), d_key=d_key, d_value=d_value, bf16=bf16)
        shape = rng.random()
        if shape < 0.2:     # one token
            c.update(n_streams=_log_int(rng, 1, 128), seg_len=1)
        elif shape < 0.6:   # segments
            c.update(n_streams=_log_int(rng, 1, 64), seg_len=_log_int(rng, 2, 128))
        else:               # long texts
            c.update(n_streams=_log_int(rng, 1, 8), seg_len=_log_int(rng, 129, 4096 if bf16 else 1024))
        c.update(ragged=int(rng.random() < 0.4), state=rng.randint(0, 1), train=int(c["seg_len"] > 1 and rng.random() < 0.5))
        return c
    if kind == "norm":
        d_key = rng.choice((32, 64, 64, 128, 2 * rng.randint(3, 64)))
        heads = _log_int(rng, 1, 16)
        return dict(kind=kind, n_rows=_log_int(rng, 1, 12000), n_head=heads, n_head_k=rng.choice((heads, 1, max(1, heads // 4))),
                    d_key=d_key, d_rot=rng.choice((d_key, d_key, d_key // 4 * 2)), adjacent=rng.randint(0, 1),
                    bf16=int(rng.random() < 0.7), far=rng.randint(0, 1), ragged=rng.randint(0, 1), train=rng.randint(0, 1))
    symbols = rng.choice((256, _log_int(rng, 100, 16384), _log_int(rng, 1024, 16384)))
    bf16 = rng.randint(0, 1)
    return dict(kind=kind, n_rows=_log_int(rng, 1, 2000), n_symbols=symbols, n_top=_log_int(rng, 1, min(100, symbols)),
                temperature=rng.choice((1.0, 1.0, 2.0, rng.uniform(0.5, 4.0))), teacher=rng.choice((1.0, 0.5, rng.uniform(0.1, 0.9))),
                bf16=bf16, grad_bf16=1 if bf16 else rng.randint(0, 1), ragged=rng.randint(0, 1), apart=rng.randint(0, 1))


# ---------------------------------------------------------------- inputs

def _type(bf16):
    return torch.bfloat16 if bf16 else torch.float32


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _prepare_linear(c, seed):
    B, H, dk, dv, T, kind = c["n_streams"], c["n_head"], c["d_key"], c["d_value"], c["seg_len"], _type(c["bf16"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (_normal(g, T * B, H * d, dtype=kind) for d in (dk, dk, dv))
    # half-lives from a few symbols to some thousand: what heads of one layer are given; every seed its own
    spread = torch.rand(H, generator=g, device="cuda", dtype=torch.float64)
    decay = (1 - 2.0 ** -(1 + 11 * (torch.arange(H, device="cuda") + spread) / H)).float()
    state = _normal(g, B, H, dk, dv) if c["state"] else None
    length = None
    if c["ragged"]:
        length = torch.randint(0, T + 1, (B,), generator=g, device="cuda").int()
        length[0] = T
        behind = (torch.arange(T, device="cuda")[:, None] >= length).reshape(T * B, 1)
        q, k, v = (torch.where(behind, float("nan"), x) for x in (q, k, v))
    s = dict(c, q=q, k=k, v=v, decay=decay.cpu(), rate=decay.double().log(), state_in=state, length=length, scale=dk ** -0.5)
    if c["train"]:
        s["dout"] = _normal(g, T * B, H * dv, dtype=kind)
        s["dstate"] = _normal(g, B, H, dk, dv) if c["state"] else None
    return s


def _prepare_norm(c, seed):
    N, H, Hk, d, kind = c["n_rows"], c["n_head"], c["n_head_k"], c["d_key"], _type(c["bf16"])
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k = (_normal(g, N, h * d, dtype=kind) for h in (H, Hk))
    gain_q, gain_k = (1 + 0.2 * _normal(g, d) for _ in range(2))
    first = int(torch.randint(0, 2 ** 30 if c["far"] else 4096, (1,), generator=g, device="cuda"))
    pos = (first + torch.arange(N, device="cuda")).int()
    if c["ragged"]:
        behind = torch.rand(N, generator=g, device="cuda") < 0.1
        pos[behind] = -1
        q, k = (torch.where(behind[:, None], float("nan"), x) for x in (q, k))
    s = dict(c, q=q, k=k, gain_q=gain_q, gain_k=gain_k, pos=pos, eps=1e-6, base=10000.0)
    if c["train"]:
        s.update(dq_out=_normal(g, N, H * d, dtype=kind), dk_out=_normal(g, N, Hk * d, dtype=kind))
    return s


def _prepare_distill(c, seed):
    N, V, K = c["n_rows"], c["n_symbols"], c["n_top"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    # logits of a trained model: a few likely symbols; the teacher's are like them, but not the same
    logits = 2.5 * _normal(g, N, V)
    teacher = logits + _normal(g, N, V)
    if c["ragged"]:  # the alphabet is filled up to a multiple of eight with symbols that no text has
        logits[:, V - 7:] = -math.inf
        teacher[:, V - 7:] = -1e4
    top, ids = teacher.topk(K, dim=1)
    targets = ids[:, 0].clone()
    other = torch.rand(N, generator=g, device="cuda") < 0.5
    targets[other] = torch.randint(0, max(1, V - 8), (N,), generator=g, device="cuda")[other]
    weight = torch.full((N,), 1.0 / N, device="cuda")
    if c["ragged"]:
        behind = torch.rand(N, generator=g, device="cuda") < 0.1
        weight[behind], targets[behind] = 0.0, -1
        ids[:, K - K // 4:][torch.rand(N, generator=g, device="cuda") < 0.5] = -1   # teachers that sent fewer
        ids[behind] = -1
        # where the student's symbol is masked, the teacher has nothing to say about it
        ids = torch.where((ids >= 0) & (logits.gather(1, ids.clamp(min=0)) == -math.inf), -1, ids)
    return dict(c, logits=logits.to(_type(c["bf16"])), ids=ids.int(), top=top.contiguous(), targets=targets.int(), weight=weight)


_PREPARE = {"linear": _prepare_linear, "norm": _prepare_norm, "distill": _prepare_distill}


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, seed)


# ---------------------------------------------------------------- the operators in their plain form

def _heads(x, s, d, behind):
    """[T * B][H * d] of any type as fp32 [B][H][T][d], zeros behind a stream's end"""
    T, B, H = s["seg_len"], s["n_streams"], s["n_head"]
    x = torch.where(behind, 0, x).float() if behind is not None else x.float()
    return x.view(T, B, H, d).permute(1, 2, 0, 3)


def _rows(x, like, behind):
    B, H, T, d = x.shape
    x = x.permute(2, 0, 1, 3).reshape(T * B, H * d)
    return (torch.where(behind, 0, x) if behind is not None else x).to(like.dtype)


def _plain_linear(s):
    B, H, dk, dv, T = s["n_streams"], s["n_head"], s["d_key"], s["d_value"], s["seg_len"]
    t = torch.arange(T, device="cuda")
    length = s["length"].long() if s["length"] is not None else torch.full((B,), T, device="cuda")
    behind = (t[:, None] >= length).reshape(T * B, 1) if s["length"] is not None else None
    q, k, v = _heads(s["q"], s, dk, behind), _heads(s["k"], s, dk, behind), _heads(s["v"], s, dv, behind)
    rate = s["rate"]
    apart = t[:, None] - t
    falls = torch.where(apart >= 0, torch.exp(rate[:, None, None] * apart), 0).float() * s["scale"]  # [H][T][T]
    since = torch.exp(rate[:, None] * (t + 1)).float()[..., None] * s["scale"]                        # [H][T][1]
    # weight of a row in the state behind the stream's last one, [B][H][T][1], and of the state before it
    left = length[:, None, None] - 1 - t
    until = torch.where(left >= 0, torch.exp(rate[:, None] * left), 0).float()[..., None]
    whole = torch.exp(rate * length[:, None]).float()[..., None, None]
    p = q @ k.transpose(2, 3) * falls
    out, state = p @ v, (until * k).transpose(2, 3) @ v
    if s["state"]:
        out, state = out + since * (q @ s["state_in"]), state + whole * s["state_in"]
    got = {"out": _rows(out, s["q"], behind), "state": state}
    if s["train"]:
        do = _heads(s["dout"], s, dv, behind)
        dp = do @ v.transpose(2, 3) * falls
        dq, dk_, dv_, dstate = dp @ k, dp.transpose(2, 3) @ q, p.transpose(2, 3) @ do, (since * q).transpose(2, 3) @ do
        if s["state"]:
            dq, dk_ = dq + since * (do @ s["state_in"].transpose(2, 3)), dk_ + until * (v @ s["dstate"].transpose(2, 3))
            dv_, dstate = dv_ + until * (k @ s["dstate"]), dstate + whole * s["dstate"]
        got.update(dq=_rows(dq, s["q"], behind), dk=_rows(dk_, s["q"], behind), dv=_rows(dv_, s["q"], behind), dstate_in=dstate)
    return got


def _turned(x, cos, sin, s):
    """The pairs of the first d_rot values turned: x [N][h][d] in fp32, cos and sin [N][1][d_rot / 2]"""
    r = s["d_rot"]
    if s["adjacent"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., r:]), -1)


def _plain_norm(s):
    N, d = s["n_rows"], s["d_key"]
    behind = (s["pos"] < 0)[:, None]
    rate = s["base"] ** -(torch.arange(0, s["d_rot"], 2, device="cuda", dtype=torch.float64) / max(1, s["d_rot"]))
    angle = s["pos"].double()[:, None, None] * rate
    cos, sin = angle.cos().float(), angle.sin().float()

    def forward(x, gain):
        x = torch.where(behind, 0, x).float().view(N, -1, d)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"])
        return x * r, r, _turned(x * r * gain, cos, sin, s)

    def back(hat, r, gain, dy):
        u = _turned(torch.where(behind, 0, dy).float().view(N, -1, d), cos, -sin, s)
        w = u * gain
        return r * (w - hat * (w * hat).mean(-1, keepdim=True)), (u * hat).sum((0, 1))

    kind = s["q"].dtype
    hat_q, r_q, y_q = forward(s["q"], s["gain_q"])
    hat_k, r_k, y_k = forward(s["k"], s["gain_k"])
    got = {"q": y_q.reshape(N, -1).to(kind), "k": y_k.reshape(N, -1).to(kind)}
    if s["train"]:
        dq, dgain_q = back(hat_q, r_q, s["gain_q"], s["dq_out"])
        dk, dgain_k = back(hat_k, r_k, s["gain_k"], s["dk_out"])
        got.update(dq=dq.reshape(N, -1).to(kind), dk=dk.reshape(N, -1).to(kind), dgain_q=dgain_q, dgain_k=dgain_k)
    return got


def _plain_softmax(z):
    """(softmax, log of the sum of exponentials) of fp32 rows"""
    m = z.max(1, keepdim=True).values
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    return e / total, m + torch.log(total)


def _plain_distill(s):
    z, tau, share = s["logits"].float(), s["temperature"], s["teacher"]
    ids, targets = s["ids"].long(), s["targets"].long()
    N, V = z.shape
    there = ids >= 0
    any_there = there.any(1, keepdim=True)
    e = torch.where(there, torch.exp((s["top"] - torch.where(there, s["top"], -1e30).max(1, keepdim=True).values) / tau), 0)
    q = e / e.sum(1, keepdim=True).clamp(min=1e-30)
    soft, lse_soft = _plain_softmax(z / tau)
    hard, lse = _plain_softmax(z)
    known = (targets >= 0)[:, None]
    of_top = torch.where(there, z.gather(1, ids.clamp(min=0)) / tau - lse_soft, 0)
    log_q = torch.where(q > 0, torch.log(q.clamp(min=1e-38)), 0)
    kl = (q * (log_q - of_top)).sum(1)
    miss = torch.where(known, lse - z.gather(1, targets.clamp(min=0)[:, None]), 0)[:, 0]
    loss = (1 - share) * miss + share * tau * tau * kl
    dz = (1 - share) * torch.where(known, hard, 0) + share * tau * torch.where(any_there, soft, 0)
    dz = dz.scatter_add(1, targets.clamp(min=0)[:, None], torch.where(known, share - 1.0, 0.0))
    dz = dz.scatter_add(1, ids.clamp(min=0), -share * tau * q)
    return {"loss": loss * s["weight"], "dlogits": (dz * s["weight"][:, None]).to(_type(s["grad_bf16"]))}


# ---------------------------------------------------------------- the framework's calls

def _ptr(x):
    return None if x is None else x.data_ptr()


def _check(rc):
    if rc:
        raise RuntimeError(_package().library().nncu_last_error().decode())


def _own_linear(s):
    pkg = _package()
    lib, st = pkg.library(), torch.cuda.current_stream().cuda_stream
    if "shape" not in s:    # what a program makes once: the shape, the results' buffers, the workspace
        B, H, dk, dv = s["n_streams"], s["n_head"], s["d_key"], s["d_value"]
        s["shape"] = pkg.abi.LinearAttnShape(n_streams=B, n_head=H, d_key=dk, d_value=dv, seg_len=s["seg_len"], scale=s["scale"],
                                             dtype_bf16=s["bf16"])
        new = {"out": torch.empty_like(s["v"]), "state": torch.empty(B, H, dk, dv, device="cuda")}
        if s["train"]:
            new.update(dq=torch.empty_like(s["q"]), dk=torch.empty_like(s["k"]), dv=torch.empty_like(s["v"]),
                       dstate_in=torch.empty_like(new["state"]))
        need = C.c_size_t()
        _check(lib.nncu_linear_attention_workspace(C.byref(s["shape"]), s["train"], C.byref(need)))
        s.update(new=new, need=need.value, room=torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda"))
    shape, new, decay = C.byref(s["shape"]), s["new"], s["decay"].data_ptr()
    q, k, v, length, state_in = (_ptr(s[n]) for n in ("q", "k", "v", "length", "state_in"))
    _check(lib.nncu_linear_attention_forward(shape, q, k, v, decay, length, state_in, _ptr(new["out"]), _ptr(new["state"]),
                                             _ptr(s["room"]), s["need"], st))
    if s["train"]:
        _check(lib.nncu_linear_attention_backward(shape, q, k, v, decay, length, state_in, _ptr(s["dout"]), _ptr(s["dstate"]),
                                                  _ptr(new["dq"]), _ptr(new["dk"]), _ptr(new["dv"]), _ptr(new["dstate_in"]),
                                                  _ptr(s["room"]), s["need"], st))
    return new


def _own_norm(s):
    pkg = _package()
    lib, st = pkg.library(), torch.cuda.current_stream().cuda_stream
    if "shape" not in s:
        s["shape"] = pkg.abi.QkNormShape(n_rows=s["n_rows"], n_head=s["n_head"], n_head_k=s["n_head_k"], d_key=s["d_key"],
                                         d_rot=s["d_rot"], adjacent=s["adjacent"], eps=s["eps"], rope_base=s["base"],
                                         dtype_bf16=s["bf16"])
        s["new"] = {n: torch.empty_like(s[n]) for n in ("q", "k")}
        if s["train"]:
            s["new"].update(dq=torch.empty_like(s["q"]), dk=torch.empty_like(s["k"]), dgain_q=torch.empty_like(s["gain_q"]),
                            dgain_k=torch.empty_like(s["gain_k"]))
            need = C.c_size_t()
            _check(lib.nncu_qk_norm_rope_workspace(C.byref(s["shape"]), C.byref(need)))
            s.update(need=need.value, room=torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda"))
    shape, new = C.byref(s["shape"]), s["new"]
    q, k, gain_q, gain_k, pos = (_ptr(s[n]) for n in ("q", "k", "gain_q", "gain_k", "pos"))
    _check(lib.nncu_qk_norm_rope_forward(shape, q, k, gain_q, gain_k, pos, _ptr(new["q"]), _ptr(new["k"]), st))
    if s["train"]:
        _check(lib.nncu_qk_norm_rope_backward(shape, q, k, gain_q, gain_k, pos, _ptr(s["dq_out"]), _ptr(s["dk_out"]),
                                              _ptr(new["dq"]), _ptr(new["dk"]), _ptr(new["dgain_q"]), _ptr(new["dgain_k"]),
                                              _ptr(s["room"]), s["need"], st))
    return new


def _own_distill(s):
    pkg = _package()
    lib, st = pkg.library(), torch.cuda.current_stream().cuda_stream
    if "shape" not in s:
        N, V = s["n_rows"], s["n_symbols"]
        s["shape"] = pkg.abi.DistillShape(n_rows=N, n_symbols=V, n_top=s["n_top"], temperature=s["temperature"],
                                          teacher_share=s["teacher"], logits_bf16=s["bf16"], grad_bf16=s["grad_bf16"])
        s["new"] = {"loss": torch.empty(N, device="cuda"), "dlogits": torch.empty(N, V, device="cuda", dtype=_type(s["grad_bf16"]))}
        s["lse"] = torch.empty(N, 2, device="cuda")
    shape, new = C.byref(s["shape"]), s["new"]
    z, ids, top, targets, weight = (_ptr(s[n]) for n in ("logits", "ids", "top", "targets", "weight"))
    if s["apart"]:
        _check(lib.nncu_distill_forward(shape, z, ids, top, targets, weight, _ptr(new["loss"]), _ptr(s["lse"]), st))
        _check(lib.nncu_distill_backward(shape, z, ids, top, targets, weight, _ptr(s["lse"]), _ptr(new["dlogits"]), st))
    else:
        _check(lib.nncu_distill_gradient(shape, z, ids, top, targets, weight, _ptr(new["loss"]), _ptr(new["dlogits"]), st))
    return new


_PLAIN = {"linear": _plain_linear, "norm": _plain_norm, "distill": _plain_distill}
_OWN = {"linear": _own_linear, "norm": _own_norm, "distill": _own_distill}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


# ---------------------------------------------------------------- the operators' definitions in 64 bits

def _exact_linear(s):
    """Token by token: the state's recurrence, and its adjoint from the last token to the first"""
    B, H, dk, dv, T = s["n_streams"], s["n_head"], s["d_key"], s["d_value"], s["seg_len"]
    q, k, v = (s[n].double().view(T, B, H, -1) for n in ("q", "k", "v"))
    length = [T] * B if s["length"] is None else s["length"].tolist()
    at = torch.tensor(length, device="cuda")
    decay = s["decay"].cuda().double()[:, None, None]
    zero = torch.zeros(B, H, dk, dv, device="cuda", dtype=torch.float64)
    state = s["state_in"].double().clone() if s["state"] else zero.clone()
    out = torch.zeros(T, B, H, dv, device="cuda", dtype=torch.float64)
    q, k, v = (torch.nan_to_num(x, nan=0.0) for x in (q, k, v))
    outer = lambda a, b: a[..., :, None] * b[..., None, :]  # noqa: E731
    dot = lambda a, m: (a[..., None, :] @ m)[..., 0, :]  # noqa: E731
    lives = lambda t: (t < at)[:, None, None, None]  # noqa: E731
    do = s["dout"].double().view(T, B, H, dv) if s["train"] else None
    dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(T):
        state = torch.where(lives(t), decay * state + outer(k[t], v[t]), state)
        out[t] = torch.where(lives(t)[..., 0], s["scale"] * dot(q[t], state), 0)
        if s["train"]:
            dq[t] = torch.where(lives(t)[..., 0], s["scale"] * dot(do[t], state.transpose(2, 3)), 0)
    got = {"out": out.view(T * B, -1), "state": state}
    if s["train"]:
        grad = s["dstate"].double().clone() if s["state"] else zero.clone()
        for t in reversed(range(T)):
            live = lives(t)
            total = grad + s["scale"] * outer(q[t], do[t])
            dk_[t] = torch.where(live[..., 0], dot(v[t], total.transpose(2, 3)), 0)
            dv_[t] = torch.where(live[..., 0], dot(k[t], total), 0)
            grad = torch.where(live, decay * total, grad)
        got.update(dq=dq.view(T * B, -1), dk=dk_.view(T * B, -1), dv=dv_.view(T * B, -1), dstate_in=grad)
    return got


def _exact_norm(s):
    """Pairs as complex numbers, gradients by differentiation"""
    N, d, r = s["n_rows"], s["d_key"], s["d_rot"]
    live = (s["pos"] >= 0)[:, None, None]
    step = torch.tensor([s["base"] ** (-2.0 * i / r) for i in range(r // 2)], device="cuda", dtype=torch.float64)
    angle = s["pos"].double()[:, None, None] * step
    turn = torch.complex(angle.cos(), angle.sin())

    def one(x, gain):
        x = torch.where(live, x.view(N, -1, d), 0).double().requires_grad_()
        gain = gain.double().requires_grad_()
        n = x / (x.square().sum(-1, keepdim=True) / d + s["eps"]).sqrt() * gain
        pair = n[..., :r].unflatten(-1, (r // 2, 2)) if s["adjacent"] else n[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        pair = pair if s["adjacent"] else pair.transpose(-1, -2)
        return x, gain, torch.cat((pair.flatten(-2), n[..., r:]), -1)

    got = {}
    for n in ("q", "k"):
        x, gain, y = one(s[n], s["gain_" + n])
        got[n] = torch.where(live, y, 0).reshape(N, -1).detach()
        if s["train"]:
            dy = torch.where(live, s["d%s_out" % n].view(N, -1, d), 0).double()
            dx, got["dgain_" + n] = torch.autograd.grad(y, (x, gain), dy)
            got["d" + n] = torch.where(live, dx, 0).reshape(N, -1)
    return got


def _exact_distill(s):
    """The loss from its definition, its gradient by differentiation"""
    z = s["logits"].double().requires_grad_()
    tau, share, ids, targets = s["temperature"], s["teacher"], s["ids"].long(), s["targets"].long()
    log_hard, log_soft = torch.log_softmax(z, 1), torch.log_softmax(z / tau, 1)
    there, known = ids >= 0, targets >= 0
    log_q = torch.log_softmax(torch.where(there, s["top"].double() / tau, -1e30), 1)
    q = torch.where(there, log_q.exp(), 0)
    kl = torch.where(there, q * (log_q - log_soft.gather(1, ids.clamp(min=0))), 0).sum(1)
    miss = torch.where(known, -log_hard.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0)
    loss = s["weight"].double() * ((1 - share) * miss + share * tau ** 2 * kl)
    return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss.sum(), z)[0]}


_EXACT = {"linear": _exact_linear, "norm": _exact_norm, "distill": _exact_distill}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "linear":
        rows, dk, dv, e = c["n_streams"] * c["n_head"] * c["seg_len"], c["d_key"], c["d_value"], 2 if c["bf16"] else 4
        states = 4 * c["n_streams"] * c["n_head"] * dk * dv
        bytes_, flops = e * rows * (2 * dk + 2 * dv) + states * (1 + c["state"]), 4 * rows * dk * dv
        if c["train"]:  # the forward results are outputs of the step, the inputs count once
            bytes_ += e * rows * (2 * dk + 2 * dv) + states * (1 + c["state"])
            flops += 10 * rows * dk * dv
        return {"bytes": bytes_, "flops": flops}
    if c["kind"] == "norm":
        values = c["n_rows"] * (c["n_head"] + c["n_head_k"]) * c["d_key"]
        e = 2 if c["bf16"] else 4
        return {"bytes": e * values * (4 if c["train"] else 2) + 4 * c["n_rows"], "flops": values * (30 if c["train"] else 10)}
    values = c["n_rows"] * c["n_symbols"]
    return {"bytes": values * ((2 if c["bf16"] else 4) + (2 if c["grad_bf16"] else 4)) + 8 * c["n_rows"] * c["n_top"],
            "flops": 10 * values}
