"""What the operators around attention cost: rotary positions with several axes,
norms of queries and keys with that rotation in the same pass, and attention
with its backward pass.

``listed()`` names the measured cases and ``draw()`` gives more of their
ranges.  ``run()`` computes a case in its plain form (elementary torch
operations in FP32), or with ``own`` set makes the calls a user makes of
``b200_pisa``.  ``exact()`` gives the same outputs from the definitions in
FP64.

A case is a dict of

* ``op``: "rope", "norm_rope", "attention" or "layer" (norm and rotation, then
  attention);
* ``pass``: "forward"; "backward" (attention only: gradients from what the
  forward pass saved); or "step" (outputs and gradients through autograd);
* ``b, hq, hk, tq, tk, d, dtype``: sizes and type; ``fused`` puts q and k into
  one [B,T,3,H,D] projection instead of separate [B,T,H,D] storage;
* ``axes`` ("44,42,42"), ``gh, gw`` (raster the positions walk), ``far`` (offset
  of the first axis' positions), ``interleaved``, ``weights`` (type of the norm
  weights) for the rotation;
* ``causal`` and ``lens`` (key lengths of the batch, "" for none) for attention.
"""
import math
import pathlib
import sys

import torch

_PACKAGE = str(pathlib.Path(__file__).resolve().parents[1] / "comfyui-rdna35-attention_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
THETA = 10000.0
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def _rope_case(name, op, direction, b, hq, hk, t, d, dtype, axes, gh, gw, interleaved, fused=False, far=0,
               weights="bf16"):
    return {"name": name, "op": op, "pass": direction, "b": b, "hq": hq, "hk": hk, "tq": t, "tk": t, "d": d,
            "dtype": dtype, "axes": axes, "gh": gh, "gw": gw, "interleaved": interleaved, "fused": fused, "far": far,
            "weights": weights}


def _attention_case(name, direction, b, hq, hk, tq, tk, d, dtype, causal=False, lens=""):
    return {"name": name, "op": "attention", "pass": direction, "b": b, "hq": hq, "hk": hk, "tq": tq, "tk": tk, "d": d,
            "dtype": dtype, "causal": causal, "lens": lens}


def listed():
    layer = _rope_case("layer_step_4096", "layer", "step", 1, 16, 4, 4096, 128, "bf16", "44,42,42", 64, 64, False)
    layer.update(causal=False, lens="")
    return [
        # the fixed-block benchmark node's default sizes: the smallest call, where latency counts
        _attention_case("attn_bwd_node_default", "backward", 1, 4, 4, 128, 128, 64, "f16"),
        # self-attention of a 1536-pixel image (96 x 96 tokens), two images: the largest
        _attention_case("attn_bwd_self_9216", "backward", 2, 16, 16, 9216, 9216, 128, "bf16"),
        # narrow heads and an odd length, as the small image models have them
        _attention_case("attn_bwd_d40_4095", "backward", 2, 8, 8, 4095, 4095, 40, "f16"),
        # image tokens that attend to a padded batch of prompts, one of them empty
        _attention_case("attn_step_prompts_512", "step", 4, 16, 16, 9216, 512, 128, "bf16",
                        lens="512,333,77,0"),
        # a causal model with shared key/value heads, one token past a tile
        _attention_case("attn_step_causal_2049", "step", 1, 40, 8, 2049, 2049, 128, "bf16", causal=True),
        # queries and keys of one 1536-pixel image in front of its attention
        _rope_case("norm_rope_image_9216", "norm_rope", "forward", 1, 16, 16, 9216, 128, "bf16", "44,42,42", 96, 96,
                   False),
        # one new token
        _rope_case("norm_rope_one_token", "norm_rope", "forward", 1, 16, 16, 1, 128, "bf16", "128", 1, 1, True, far=4097),
        # a training step of the same in front of the interleaved 56-head projection
        _rope_case("norm_rope_step_9170", "norm_rope", "step", 1, 56, 56, 9170, 128, "bf16", "32,48,48", 70, 131, True,
                   fused=True, weights="f32"),
        # the queries of a video of 21 frames of 30 x 52 tokens
        _rope_case("rope_video_32760", "rope", "forward", 1, 40, 40, 32760, 128, "bf16", "44,42,42", 30, 52, True),
        # a prompt's tokens far along the axis, narrow heads of which a part is rotated, and their gradient
        _rope_case("rope_step_far_77", "rope", "step", 2, 8, 8, 77, 64, "f16", "24,12,12", 7, 11, False, far=1000003),
        # norm, rotation and attention of one layer with shared key/value heads, and all gradients
        layer,
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


#: (query, key) pairs over all heads of the largest listed case
MOST_PAIRS = 2 * 16 * 9216 * 9216


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "norm_rope", "norm_rope", "rope", "layer"])
    d = rng.choice([32, 40, 64, 64, 80, 96, 120, 128, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    hk = _log(rng, 1, 24)
    group = rng.choice([1, 1, 2, 4, 7])
    b = _log(rng, 1, 6)
    if op in ("attention", "layer"):
        tq = _log(rng, 64, 9300)
        tk = tq if op == "layer" or rng.random() < 0.5 else _log(rng, 2, 9300)
        if op == "attention" and rng.random() < 0.1:
            tq = _log(rng, 1, 64)
        while b * hk * group * tq * tk > MOST_PAIRS:
            if b > 1:
                b -= 1
            elif group > 1:
                group = 1
            else:
                hk -= 1
    if op == "attention":
        lens = ""
        if b > 1 and rng.random() < 0.5:
            lens = ",".join([str(tk)] + [str(rng.choice([0, 1 + rng.randrange(tk), 1 + rng.randrange(tk)]))
                                         for _ in range(b - 1)])
        case = _attention_case("", rng.choice(["backward", "step"]), b, hk * group, hk, tq, tk, d, dtype,
                               causal=rng.random() < 0.3 and tq <= tk, lens=lens)
    else:
        t = tq if op == "layer" else _log(rng, 1, 33000)
        while b * hk * (group + 1) * t * d > 2 * 56 * 9170 * 128:
            b, hk = (b - 1, hk) if b > 1 else (b, hk - 1) if hk > 1 else (b, hk)
            t = t if b * hk > 1 else max(1, t // 2)
        if op != "layer":
            dtype = rng.choice(["bf16", "f16", "f32"])
        rotated = rng.choice([d, d, d // 16 * 8])
        third = rotated // 3 // 2 * 2
        axes = rng.choice([str(rotated), "%d,%d,%d" % (rotated - 2 * third, third, third)])
        gw = _log(rng, 1, 131)
        gh = _log(rng, 1, 131)
        case = _rope_case("", op, "step" if op == "layer" else rng.choice(["forward", "step"]), b, hk * group, hk, t, d,
                          dtype, axes, gh, gw, rng.random() < 0.5, fused=group == 1 and rng.random() < 0.5,
                          far=rng.choice([0, 0, _log(rng, 1, 2000000)]),
                          weights=dtype if op == "layer" else rng.choice([dtype, "f32"]))
        if op == "layer":
            case.update(causal=rng.random() < 0.5, lens="")
    del case["name"]
    return case


# ------------------------------------------------------------------ the inputs
def _normal(gen, shape, scale, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _heads(storage):
    """The [B,H,T,D] view of [B,T,H,D] storage."""
    return storage.permute(0, 2, 1, 3)


def _positions(case):
    """Integer positions [T,A] of tokens that walk a raster, frame after frame."""
    t = torch.arange(case["tq"], device="cuda")
    gh, gw = case["gh"], case["gw"]
    axes = len(case["axes"].split(","))
    if axes == 1:
        return (t + case["far"])[:, None]
    return torch.stack([t // (gh * gw) + case["far"], t // gw % gh, t % gw], dim=1)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, hq, hk, tq, tk, d = (case[n] for n in ("b", "hq", "hk", "tq", "tk", "d"))
    s = {}
    if case["op"] == "rope":
        s["q"] = _heads(_normal(gen, (b, tq, hq, d), 1.0, dt))
    elif case.get("fused"):
        qkv = _normal(gen, (b, tq, 3, hq, d), 1.0, dt)
        s["q"], s["k"], s["v"] = (_heads(qkv[:, :, i]) for i in range(3))
    else:
        s["q"] = _heads(_normal(gen, (b, tq, hq, d), 1.0, dt))
        s["k"] = _heads(_normal(gen, (b, tk, hk, d), 1.0, dt))
        s["v"] = _heads(_normal(gen, (b, tk, hk, d), 1.0, dt))
    if case["op"] in ("norm_rope", "layer"):
        wt = DTYPES[case["weights"]]
        s["wq"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(wt)
        s["wk"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(wt)
    if "axes" in case:
        s["pos"] = _positions(case)
    if case["op"] in ("attention", "layer"):
        # queries and keys of one direction in common, so that rows have keys that stand out
        common = torch.randn(d, generator=gen, device="cuda")
        for n in ("q", "k"):
            s[n] += (0.5 * common).to(dt)
        if case["pass"] != "forward":
            s["dout"] = _heads(_normal(gen, (b, tq, hq, d), 1.0, dt))
        s["lens"] = None
        if case["lens"]:
            s["lens"] = torch.tensor([int(x) for x in case["lens"].split(",")], dtype=torch.int32, device="cuda")
    elif case["pass"] == "step":
        s["dq"] = _heads(_normal(gen, (b, tq, hq, d), 1.0, dt))
        if case["op"] == "norm_rope":
            s["dk"] = _heads(_normal(gen, (b, tk, hk, d), 1.0, dt))
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "attention" and case["pass"] == "backward":
        # what the forward pass left
        out, state["lse"] = _plain_attention(state["q"], state["k"], state["v"], _scale(case), case["causal"],
                                             state["lens"])
        state["out"] = _heads(out.to(DTYPES[case["dtype"]]).permute(0, 2, 1, 3).contiguous())
    if case["pass"] == "step":
        for n in ("q", "k", "v", "wq", "wk"):
            if n in state and (n != "v" or case["op"] in ("attention", "layer")):
                state[n] = state[n].detach().requires_grad_()
    return state


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


def _axes(case):
    return tuple(int(x) for x in case["axes"].split(","))


# ------------------------------------------------------------------ plain forms
def _plain_angles(pos, axes):
    """cos and sin [T,1,R/2] in FP32 of angles computed in FP64."""
    cols = [pos[:, a, None].double() * THETA ** (-torch.arange(0, n, 2, device="cuda").double() / n)
            for a, n in enumerate(axes)]
    angle = torch.cat(cols, dim=1)
    return angle.cos().float(), angle.sin().float()


def _plain_rotate(x, cos, sin, interleaved):
    """x [B,H,T,D] FP32 with its first 2*cos.shape[-1] columns rotated."""
    r = 2 * cos.shape[-1]
    rot = x[..., :r]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = rot[..., : r // 2], rot[..., r // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y, x[..., r:]), dim=-1)


def _plain_norm(x, w):
    rstd = torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS)
    return x * rstd * w, rstd


def _plain_norm_backward(dz, x, rstd, w):
    xh = x * rstd
    dw = (dz * xh).sum(dim=(0, 1, 2))
    g = dz * w
    return rstd * (g - xh * (g * xh).mean(dim=-1, keepdim=True)), dw


def _plain_mask(q, k, causal, lens):
    """Which keys each query sees, [B|1,1,Tq,Tk], or None for all."""
    tq, tk = q.shape[2], k.shape[2]
    keep = None
    if causal:
        keep = torch.ones((tq, tk), dtype=torch.bool, device="cuda").tril(tk - tq)[None, None]
    if lens is not None:
        short = (torch.arange(tk, device="cuda") < lens[:, None])[:, None, None]
        keep = short if keep is None else keep & short
    return keep


def _plain_scores(q, k, scale, keep):
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    return s if keep is None else s.masked_fill_(~keep, -math.inf)


def _plain_wide(q, k, v):
    group = q.shape[1] // k.shape[1]
    q, k, v = q.float(), k.float(), v.float()
    return (q, k, v) if group == 1 else (q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1))


def _plain_attention(q, k, v, scale, causal, lens):
    """(out FP32, lse FP32); rows without a key give 0 and -inf."""
    keep = _plain_mask(q, k, causal, lens)
    q, k, v = _plain_wide(q, k, v)
    s = _plain_scores(q, k, scale, keep)
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (total.log() + top).squeeze(-1)


def _plain_attention_backward(dout, q, k, v, out, lse, scale, causal, lens):
    heads, kv_heads = q.shape[1], k.shape[1]
    keep = _plain_mask(q, k, causal, lens)
    q, k, v = _plain_wide(q, k, v)
    dout = dout.float()
    delta = (dout * out.float()).sum(dim=-1, keepdim=True)
    lse = torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None]
    p = _plain_scores(q, k, scale, keep).sub_(lse).exp_()
    dv = torch.matmul(p.transpose(-1, -2), dout)
    ds = torch.matmul(dout, v.transpose(-1, -2)).sub_(delta).mul_(p)
    del p
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(-1, -2), q) * scale
    if heads != kv_heads:
        dk, dv = (x.unflatten(1, (kv_heads, heads // kv_heads)).sum(dim=2) for x in (dk, dv))
    return dq, dk, dv


def _run_plain(s):
    case = s["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "attention":
        q, k, v = (s[n].detach() for n in "qkv")
        if case["pass"] == "backward":
            grads = _plain_attention_backward(s["dout"], q, k, v, s["out"], s["lse"], _scale(case), case["causal"],
                                              s["lens"])
            return tuple(x.to(dt) for x in grads)
        out, lse = _plain_attention(q, k, v, _scale(case), case["causal"], s["lens"])
        grads = _plain_attention_backward(s["dout"], q, k, v, out, lse, _scale(case), case["causal"], s["lens"])
        return tuple(x.to(dt) for x in (out, *grads))
    cos, sin = _plain_angles(s["pos"], _axes(case))
    inter = case["interleaved"]
    q = s["q"].detach().float()
    if case["op"] == "rope":
        y = _plain_rotate(q, cos, sin, inter).to(dt)
        if case["pass"] == "forward":
            return y
        return y, _plain_rotate(s["dq"].float(), cos, -sin, inter).to(dt)
    k = s["k"].detach().float()
    wq, wk = s["wq"].detach(), s["wk"].detach()
    zq, rq = _plain_norm(q, wq.float())
    zk, rk = _plain_norm(k, wk.float())
    yq, yk = _plain_rotate(zq, cos, sin, inter), _plain_rotate(zk, cos, sin, inter)
    if case["pass"] == "forward":
        return yq.to(dt), yk.to(dt)
    if case["op"] == "layer":
        v = s["v"].detach()
        out, lse = _plain_attention(yq, yk, v, _scale(case), case["causal"], s["lens"])
        dyq, dyk, dv = _plain_attention_backward(s["dout"], yq, yk, v, out, lse, _scale(case), case["causal"], s["lens"])
    else:
        dyq, dyk = s["dq"].float(), s["dk"].float()
    dq, dwq = _plain_norm_backward(_plain_rotate(dyq, cos, -sin, inter), q, rq, wq.float())
    dk, dwk = _plain_norm_backward(_plain_rotate(dyk, cos, -sin, inter), k, rk, wk.float())
    grads = (dq.to(dt), dk.to(dt), dwq.to(wq.dtype), dwk.to(wk.dtype))
    if case["op"] == "layer":
        return (out.to(dt), dv.to(dt), *grads)
    return (yq.to(dt), yk.to(dt), *grads)


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    import b200_pisa

    case = s["case"]
    if case["op"] == "attention":
        if case["pass"] == "backward":
            return b200_pisa.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"],
                                                causal=case["causal"], key_lengths=s["lens"])
        out = b200_pisa.attention(s["q"], s["k"], s["v"], causal=case["causal"], key_lengths=s["lens"])
        return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))
    rotation = dict(theta=THETA, interleaved=case["interleaved"])
    if case["op"] == "rope":
        y = b200_pisa.axial_rope(s["q"], s["pos"], _axes(case), **rotation)
        if case["pass"] == "forward":
            return y
        return y.detach(), torch.autograd.grad(y, s["q"], s["dq"])[0]
    if case["op"] == "layer":
        out = b200_pisa.norm_rope_attention(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["pos"], _axes(case), eps=EPS,
                                            causal=case["causal"], key_lengths=s["lens"], **rotation)
        dv, *grads = torch.autograd.grad(out, [s[n] for n in ("v", "q", "k", "wq", "wk")], s["dout"])
        return (out.detach(), dv, *grads)
    q, k = b200_pisa.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], _axes(case), eps=EPS, **rotation)
    if case["pass"] == "forward":
        return q, k
    return (q.detach(), k.detach(),
            *torch.autograd.grad((q, k), [s[n] for n in ("q", "k", "wq", "wk")], (s["dq"], s["dk"])))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Unmasked (query, key) pairs of one head, summed over the batch."""
    tq, tk = case["tq"], case["tk"]
    lens = [int(x) for x in case["lens"].split(",")] if case["lens"] else [tk] * case["b"]
    if not case["causal"]:
        return sum(tq * n for n in lens)
    return sum(sum(min(max(i + tk - tq + 1, 0), n) for i in range(tq)) for n in lens)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    q = case["b"] * case["hq"] * case["tq"] * case["d"]
    k = case["b"] * case["hk"] * case["tk"] * case["d"]
    step = case["pass"] == "step"
    if case["op"] == "rope":
        return {"bytes": (4 if step else 2) * q * es, "flops": (6 if step else 3) * q}
    if case["op"] == "norm_rope":
        # forward reads q, k and writes both; the gradients read theirs and q, k again and are written
        return {"bytes": (5 if step else 2) * (q + k) * es, "flops": (25 if step else 8) * (q + k)}
    product = 2 * case["hq"] * case["d"] * _pairs(case)
    if case["op"] == "layer":
        return {"bytes": (4 * q + 4 * k) * es, "flops": 7 * product}
    if case["pass"] == "backward":
        return {"bytes": (4 * q + 4 * k) * es + 4 * q // case["d"], "flops": 5 * product}
    return {"bytes": (4 * q + 4 * k) * es, "flops": 7 * product}


# ------------------------------------------------------------------ the definitions in FP64
def _exact_rotation(case, pos):
    """The rotation as a function of x [..., T, D]: complex multiplication."""
    turn = []
    for a, n in enumerate(_axes(case)):
        for j in range(n // 2):
            turn.append(pos[:, a].double() * math.pow(THETA, -2.0 * j / n))
    angle = torch.stack(turn, dim=-1)
    unit = torch.polar(torch.ones_like(angle), angle)
    half = unit.shape[-1]

    def rotate(x, back=False):
        u = unit.conj() if back else unit
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., : 2 * half].unflatten(-1, (half, 2)).contiguous()) * u
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half: 2 * half].contiguous()) * u
            y = torch.cat((z.real, z.imag), dim=-1)
        return torch.cat((y, x[..., 2 * half:]), dim=-1)

    return rotate


def _exact_attention(q, k, v, dout, scale, causal, lens):
    """out, dq, dk, dv of FP64 q, k, v, dout, one (batch, head) at a time."""
    b, hq, tq, d = q.shape
    hk, tk = k.shape[1], k.shape[2]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for i in range(b):
        n = tk if lens is None else int(lens[i])
        if n == 0:
            continue
        for h in range(hq):
            g = h // (hq // hk)
            kk, vv = k[i, g, :n], v[i, g, :n]
            logits = (q[i, h] @ kk.T) * scale
            if causal:
                row = torch.arange(tq, device="cuda")[:, None]
                logits[torch.arange(n, device="cuda")[None, :] > row + (tk - tq)] = -math.inf
            p = torch.softmax(logits, dim=-1)
            p = torch.where(torch.isnan(p), torch.zeros_like(p), p)
            out[i, h] = p @ vv
            dp = dout[i, h] @ vv.T
            ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
            dq[i, h] = scale * (ds @ kk)
            dk[i, g, :n] += scale * (ds.T @ q[i, h])
            dv[i, g, :n] += p.T @ dout[i, h]
    return out, dq, dk, dv


def exact(case, seed):
    s = {n: x.double() if x is not None and x.is_floating_point() else x for n, x in _inputs(case, seed).items()}
    if case["op"] == "attention":
        got = _exact_attention(s["q"], s["k"], s["v"], s["dout"], _scale(case), case["causal"], s["lens"])
        return got[1:] if case["pass"] == "backward" else got
    rotate = _exact_rotation(case, s["pos"])
    if case["op"] == "rope":
        y = rotate(s["q"])
        return y if case["pass"] == "forward" else (y, rotate(s["dq"], back=True))

    def normed(x, w):
        return x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS) * w

    def gradients(x, w, dy):
        r = 1.0 / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / x.shape[-1] + EPS)
        dz = rotate(dy, back=True)
        inner = (dz * w * x).sum(dim=-1, keepdim=True) / x.shape[-1]
        return dz * w * r - x * inner * r ** 3, (dz * x * r).flatten(0, 2).sum(dim=0)

    yq, yk = rotate(normed(s["q"], s["wq"])), rotate(normed(s["k"], s["wk"]))
    if case["pass"] == "forward":
        return yq, yk
    if case["op"] == "layer":
        out, s["dq"], s["dk"], dv = _exact_attention(yq, yk, s["v"], s["dout"], _scale(case), case["causal"], s["lens"])
    dq, dwq = gradients(s["q"], s["wq"], s["dq"])
    dk, dwk = gradients(s["k"], s["wk"], s["dk"])
    return (out, dv, dq, dk, dwq, dwk) if case["op"] == "layer" else (yq, yk, dq, dk, dwq, dwk)
