"""Measured cases of the producer LM's block operators, with their plain forms.

Three operators of a decoder block that follow one another in a forward pass:

* `linear`  y = x W^T (+ bias) with W held in e4m3 with one fp32 scale per 128 x 128 block and x
  quantised on the way in, one scale per row and 128 columns; in training also the gradient of x,
  with the incoming gradient quantised the same way (W and bias are frozen).
* `norm`    stream = x + scale * gate * post_norm(branch), normed = pre_norm(stream): the end of one
  sub-block and the start of the next.  The stream is rounded to its type once, and the pre-norm
  reads what was stored; in training the gradients of every tensor.
* `rotary`  rotary positions of q and k: the first `rot` channels of each head, paired half with
  half or neighbour with neighbour, angles position * frequency; in training the gradients too.

`run` computes the plain form in 32 bits, or calls `saelens_b200.ops` when `own` is set; `exact`
evaluates the definitions in 64 bits.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
BLOCK = 128
LEAST = E4M3_MAX * torch.finfo(torch.float32).tiny  # least maximum of a block: the scale stays a normal number
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------ the cases
def _linear(name, m, k, n, bias=False, train=False, dtype="bf16"):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "bias": bias, "train": train, "dtype": dtype}


def _norm(name, b, s, d, kind="rms", one_plus=False, post=False, gate="none", scale=1.0, train=False, dtype="bf16"):
    return {"name": name, "op": "norm", "b": b, "s": s, "d": d, "kind": kind, "one_plus": one_plus, "post": post,
            "gate": gate, "scale": scale, "train": train, "dtype": dtype}


def _rotary(name, b, s, h, kv, d, rot, interleaved=False, scaling="none", first=0, train=False, dtype="bf16"):
    return {"name": name, "op": "rotary", "b": b, "s": s, "h": h, "kv": kv, "d": d, "rot": rot,
            "interleaved": interleaved, "scaling": scaling, "first": first, "train": train, "dtype": dtype}


def listed():
    return [
        # one token through the fused q/k/v projection of the Llama-3-8B preset: weight bandwidth and latency
        _linear("linear qkv, one token", 1, 4096, 6144),
        # one token of each of 24 sequences through that preset's down projection
        _linear("linear down, 24 tokens", 24, 14336, 4096),
        # a short ragged prompt batch through the biased q/k/v projection of the Qwen2.5-14B preset
        _linear("linear qkv, 333 tokens", 333, 5120, 7168, bias=True),
        # an activation-capture batch through the fused gate/up projection of the Llama-3-8B preset
        _linear("linear gate/up, 8192 tokens", 8192, 4096, 28672),
        # attribution through a frozen up projection: the output and the gradient of its input
        _linear("linear up with gradient", 2048, 4096, 14336, train=True),
        # one token between two sub-blocks of the Llama-3-8B preset: latency
        _norm("norm, one token", 1, 1, 4096),
        # a capture batch of that preset
        _norm("norm, 8192 tokens", 8, 1024, 4096),
        # the Gemma-2-9B preset's post- and pre-norms around a ragged batch
        _norm("norm sandwich, 3 x 1365", 3, 1365, 3584, one_plus=True, post=True),
        # LayerNorm at the GPT-2 preset's width, with a gate per channel and a branch scale, trained
        _norm("norm gated with gradients", 8, 513, 768, kind="layer", post=True, gate="channel", scale=0.5,
              train=True, dtype="fp32"),
        # 64 sequences, one token each, far into a context stretched by frequency bands
        _rotary("rotary, 64 single tokens", 64, 1, 32, 8, 128, 128, scaling="llama3", first=100003),
        # a capture batch of the Llama-3-8B preset
        _rotary("rotary, 8192 tokens", 4, 2048, 32, 8, 128, 128),
        # neighbour pairs over a quarter of Gemma-2's wide heads, with gradients
        _rotary("rotary part with gradients", 2, 1023, 16, 8, 256, 64, interleaved=True, scaling="yarn", first=5,
                train=True, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "norm", "rotary"])
    train = rng.random() < 0.3
    if op == "linear":
        c = _linear("", _log(rng, 1, 4096), _log(rng, 64, 8192), _log(rng, 64, 16384), bias=rng.random() < 0.4,
                    train=train, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    elif op == "norm":
        d = _log(rng, 64, 8192)
        if rng.random() < 0.7:  # most widths are whole 16-byte vectors
            d = max(64, d // 8 * 8)
        c = _norm("", _log(rng, 1, 8), _log(rng, 1, 2048), d, kind=rng.choice(["rms", "layer"]),
                  one_plus=rng.random() < 0.3, post=rng.random() < 0.5,
                  gate=rng.choice(["none", "channel", "sequence", "token"]), scale=rng.choice([1.0, 0.25, 0.7071]),
                  train=train, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    else:
        kv = rng.choice([1, 2, 4, 8])
        d = 2 * _log(rng, 16, 128)
        rot = d if rng.random() < 0.5 else 2 * _log(rng, 4, d // 2)
        c = _rotary("", _log(rng, 1, 16), _log(rng, 1, 2048), kv * rng.choice([1, 2, 4]), kv, d, rot,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                    first=_log(rng, 1, 1000000), train=train, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    del c["name"]
    return c


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        b = e * m * k + n * k + 4 * (-(-n // BLOCK)) * (-(-k // BLOCK)) + e * m * n + (4 * n if case["bias"] else 0)
        f = 2.0 * m * n * k
        if case["train"]:  # the output's gradient read, the input's written; W is read once for both products
            b, f = b + e * (m * n + m * k), 2 * f
        return {"bytes": b, "flops": f}
    if case["op"] == "norm":
        rows, d = case["b"] * case["s"], case["d"]
        g = {"none": 0, "channel": d, "sequence": case["b"] * d, "token": rows * d}[case["gate"]]
        vectors = d * ((2 if case["kind"] == "layer" else 1) * (2 if case["post"] else 1))
        b, f = e * (4 * rows * d + g + vectors), 12.0 * rows * d
        if case["train"]:  # two gradients read, two written, and those of the gate and the vectors
            same = not (case["post"] or case["gate"] != "none" or case["scale"] != 1.0)
            b, f = b + e * ((3 if same else 4) * rows * d + g + vectors), 3 * f
        return {"bytes": b, "flops": f}
    rows = case["b"] * case["s"]
    values = rows * (case["h"] + case["kv"]) * case["d"]
    b, f = 2 * e * values + 8 * rows + 4 * case["rot"], 3.0 * values
    return {"bytes": 2 * b if case["train"] else b, "flops": 2 * f if case["train"] else f}


# ------------------------------------------------------------------------------------ the inputs
def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)


def _frequencies(rot, scaling):
    """Angle per position of each pair, in 64 bits, and the factor that the stretched context puts on
    cos and sin."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":  # positions squeezed by 4
        return f / 4.0, 1.0
    if scaling == "llama3":  # long wavelengths squeezed by 8, a ramp between, 8192 positions before
        turns = 8192.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f / 8.0 * (1 - keep) + f * keep, 1.0
    if scaling == "yarn":  # pairs that turn fewer than 1 to 32 times in 4096 positions squeezed by 16
        at = [rot * math.log(4096.0 / (t * 2 * math.pi)) / (2 * math.log(10000.0)) for t in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / 16.0 * ramp + f * (1 - ramp), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _blocks(t):
    """t [rows, columns] in 128-column blocks [rows, blocks, 128], zeros behind the last column."""
    return torch.nn.functional.pad(t, (0, -t.shape[1] % BLOCK)).view(t.shape[0], -1, BLOCK)


def _quantized_weight(gen, n, k):
    """A projection's weight in e4m3 (rows 16-byte aligned) and its scale per 128 x 128 block."""
    w = _randn(gen, n, k, std=k ** -0.5)
    w[:, :: 61] *= 4.0  # channels of larger weights, as trained projections have
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    t = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scale = t.abs().amax(dim=(1, 3)).clamp_min(LEAST) / E4M3_MAX
    t = (t / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    q = torch.zeros(n, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device="cuda")
    q[:, :k] = t.view(nb * BLOCK, kb * BLOCK)[:n, :k]
    return q[:, :k], scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 40))
    dt, train = TYPES[case["dtype"]], case["train"]
    st = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = _randn(gen, m, k)
        x[:, :: 97] *= 10.0  # the few large channels of a residual stream
        st["x"] = x.to(dt).requires_grad_(train)
        st["w"], st["w_scale"] = _quantized_weight(gen, n, k)
        st["bias"] = _randn(gen, n) if case["bias"] else None
        if train:
            st["dy"] = _randn(gen, m, n, dtype=dt, std=0.05)
        return st
    if case["op"] == "norm":
        b, s, d = case["b"], case["s"], case["d"]
        st["x"] = _randn(gen, b, s, d, dtype=dt, std=2.0)
        st["branch"] = _randn(gen, b, s, d, dtype=dt, std=0.7)
        mid = 0.0 if case["one_plus"] else 1.0
        st["w"] = _randn(gen, d, std=0.1).add(mid).to(dt)
        st["w_bias"] = _randn(gen, d, dtype=dt, std=0.1) if case["kind"] == "layer" else None
        st["post_w"] = _randn(gen, d, std=0.1).add(mid).to(dt) if case["post"] else None
        st["post_bias"] = _randn(gen, d, dtype=dt, std=0.1) if case["post"] and case["kind"] == "layer" else None
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, s, d)}[case["gate"]]
        st["gate"] = None if shape is None else _randn(gen, *shape, std=0.3).add(1.0).to(dt)
        if train:
            st["d_stream"], st["d_normed"] = _randn(gen, b, s, d, dtype=dt), _randn(gen, b, s, d, dtype=dt)
            for name in NORM_INPUTS:
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    b, s, h, kv, d = case["b"], case["s"], case["h"], case["kv"], case["d"]
    # q and k are views of the fused projection's output, as the producer LM has them
    qkv = _randn(gen, b, s, (h + 2 * kv) * d, dtype=dt)
    st["q"] = qkv[..., : h * d].view(b, s, h, d).requires_grad_(train)
    st["k"] = qkv[..., h * d : (h + kv) * d].view(b, s, kv, d).requires_grad_(train)
    starts = torch.randint(0, 1024, (b, 1), device="cuda", generator=gen) + case["first"]
    st["positions"] = starts + torch.arange(s, device="cuda")
    f, st["factor"] = _frequencies(case["rot"], case["scaling"])
    st["freq"] = f.to("cuda")
    if train:
        st["dq"], st["dk"] = _randn(gen, b, s, h, d, dtype=dt), _randn(gen, b, s, kv, d, dtype=dt)
    return st


NORM_INPUTS = ("x", "branch", "w", "w_bias", "post_w", "post_bias", "gate")
NORM_EPS = 1e-6


# ------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "rotary": _own_rotary}[op](state)
    return {"linear": _plain_linear, "norm": _plain_norm, "rotary": _plain_rotary}[op](state)


_STATUS = {}


def _status(device):
    """The program's status word of the device, kept over its calls."""
    if device not in _STATUS:
        from saelens_b200.ops import StatusWord

        _STATUS[device] = StatusWord(device)
    return _STATUS[device]


def _own_linear(st):
    from saelens_b200 import ops

    y = ops.linear_fp8(st["x"], st["w"], st["w_scale"], bias=st["bias"], status=_status(st["x"].device))
    if not st["case"]["train"]:
        return {"y": y}
    (dx,) = torch.autograd.grad(y, (st["x"],), st["dy"])
    return {"y": y, "dx": dx}


def _own_norm(st):
    from saelens_b200 import ops

    c = st["case"]
    stream, normed = ops.residual_norm(
        st["x"], st["branch"], st["w"], st["w_bias"], kind=c["kind"], eps=NORM_EPS, one_plus=c["one_plus"],
        post_weight=st["post_w"], post_bias=st["post_bias"], gate=st["gate"], scale=c["scale"])
    out = {"stream": stream, "normed": normed}
    if c["train"]:
        names = [n for n in NORM_INPUTS if st[n] is not None]
        grads = torch.autograd.grad((stream, normed), [st[n] for n in names], (st["d_stream"], st["d_normed"]))
        out.update({"d_" + n: g for n, g in zip(names, grads)})
    return out


def _own_rotary(st):
    from saelens_b200 import ops

    q, k = ops.rotary(st["q"], st["k"], st["freq"], positions=st["positions"],
                      interleaved=st["case"]["interleaved"], factor=st["factor"])
    if not st["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _plain_quantize(t):
    """Rows of t in 32 bits as the values that e4m3 with a scale per 128 columns holds.  The quotient
    t * 448 / max is rounded once where t has 16 bits (7/16 t is exact and cannot overflow), so that
    values on the border of two e4m3 neighbours fall the same way whatever the arithmetic."""
    blocks = _blocks(t)
    most = blocks.abs().amax(-1, keepdim=True).clamp_min(LEAST)
    held = (blocks * (E4M3_MAX / 1024.0) / most * 1024.0).to(torch.float8_e4m3fn).float() * (most / E4M3_MAX)
    return held.view(t.shape[0], -1)[:, : t.shape[1]]


def _plain_linear(st):
    x, dt = st["x"].detach(), st["x"].dtype
    n, k = st["w"].shape
    scale = st["w_scale"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    w = st["w"].float() * scale
    y = _plain_quantize(x.float()) @ w.T
    if st["bias"] is not None:
        y = y + st["bias"]
    out = {"y": y.to(dt)}
    if st["case"]["train"]:
        out["dx"] = (_plain_quantize(st["dy"].float()) @ w).to(dt)
    return out


def _plain_normalize(t, w, bias, case):
    if case["kind"] == "layer":
        t = t - t.mean(-1, keepdim=True)
    t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + NORM_EPS) * (1.0 + w if case["one_plus"] else w)
    return t if bias is None else t + bias


def _plain_norm(st):
    c, dt = st["case"], st["x"].dtype
    names = [n for n in NORM_INPUTS if st[n] is not None]
    v = {n: st[n].detach().float().requires_grad_(c["train"]) for n in names}
    with torch.set_grad_enabled(c["train"]):
        u = v["branch"]
        if c["post"]:
            u = _plain_normalize(u, v["post_w"], v.get("post_bias"), c)
        if "gate" in v:
            u = u * v["gate"]
        stream = v["x"] + u * c["scale"]
        stored = stream + (stream.to(dt).float() - stream).detach()  # the pre-norm reads the stored stream
        normed = _plain_normalize(stored, v["w"], v.get("w_bias"), c)
        out = {"stream": stream.detach().to(dt), "normed": normed.detach().to(dt)}
        if c["train"]:
            grads = torch.autograd.grad((stream, normed), [v[n] for n in names],
                                        (st["d_stream"].float(), st["d_normed"].float()))
            out.update({"d_" + n: g.to(dt) for n, g in zip(names, grads)})
    return out


def _plain_rotate(t, cos, sin, interleaved):
    rot, f = 2 * cos.shape[-1], t.float()
    a, b = (f[..., 0:rot:2], f[..., 1:rot:2]) if interleaved else (f[..., : rot // 2], f[..., rot // 2 : rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, f[..., rot:]), -1).to(t.dtype)


def _plain_rotary(st):
    angle = st["positions"].double()[..., None] * st["freq"]  # 64 bits: far positions
    cos = (torch.cos(angle) * st["factor"]).float()[:, :, None]
    sin = (torch.sin(angle) * st["factor"]).float()[:, :, None]
    turn = st["case"]["interleaved"]
    out = {n: _plain_rotate(st[n].detach(), cos, sin, turn) for n in ("q", "k")}
    if st["case"]["train"]:  # the transposed rotation
        out.update({n: _plain_rotate(st[n], cos, -sin, turn) for n in ("dq", "dk")})
    return out


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "rotary": _exact_rotary}[case["op"]](st)


def _e4m3(v):
    """The nearest e4m3 value (ties to even): 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    v = v.clamp(-E4M3_MAX, E4M3_MAX)
    e = torch.frexp(v)[1].clamp_min(-5) - 4
    return torch.ldexp(torch.round(torch.ldexp(v, -e)), e)


def _exact_held(t):
    cols = t.shape[1]
    t = torch.cat((t, t.new_zeros(t.shape[0], -cols % BLOCK)), 1)
    parts = []
    for c in range(0, t.shape[1], BLOCK):
        part = t[:, c : c + BLOCK]
        most = part.abs().max(dim=1, keepdim=True).values
        most = torch.where(most < LEAST, LEAST, most)
        parts.append(_e4m3(part * E4M3_MAX / most) * (most / E4M3_MAX))
    return torch.cat(parts, 1)[:, :cols]


def _exact_linear(st):
    n, k = st["w"].shape
    rows, cols = torch.arange(n, device="cuda") // BLOCK, torch.arange(k, device="cuda") // BLOCK
    w = st["w"].double() * st["w_scale"].double()[rows][:, cols]
    y = torch.einsum("mk,nk->mn", _exact_held(st["x"].detach().double()), w)
    out = {"y": y if st["bias"] is None else y + st["bias"].double()}
    if st["case"]["train"]:
        out["dx"] = torch.einsum("mn,nk->mk", _exact_held(st["dy"].double()), w)
    return out


def _exact_unit(t, layer):
    """t normalised without its vectors, and the reciprocal deviation."""
    if layer:
        t = t - t.sum(-1, keepdim=True) / t.shape[-1]
    r = 1.0 / torch.sqrt(t.square().sum(-1, keepdim=True) / t.shape[-1] + NORM_EPS)
    return t * r, r


def _exact_unit_backward(g, unit, r, layer):
    out = g - unit * (g * unit).mean(-1, keepdim=True)
    return (out - g.mean(-1, keepdim=True) if layer else out) * r


def _exact_norm(st):
    c = st["case"]
    layer, add = c["kind"] == "layer", 1.0 if c["one_plus"] else 0.0
    v = {n: st[n].detach().double() for n in NORM_INPUTS if st[n] is not None}
    u = v["branch"]
    if c["post"]:
        b_unit, b_r = _exact_unit(u, layer)
        u = b_unit * (v["post_w"] + add)
        if layer:
            u = u + v["post_bias"]
    gate = v["gate"] if "gate" in v else torch.ones((), dtype=torch.float64, device="cuda")
    stream = v["x"] + c["scale"] * gate * u
    unit, r = _exact_unit(stream.to(st["x"].dtype).double(), layer)
    normed = unit * (v["w"] + add)
    if layer:
        normed = normed + v["w_bias"]
    out = {"stream": stream, "normed": normed}
    if c["train"]:
        g = st["d_normed"].double()
        out["d_w"] = (g * unit).sum((0, 1))
        if layer:
            out["d_w_bias"] = g.sum((0, 1))
        g = st["d_stream"].double() + _exact_unit_backward(g * (v["w"] + add), unit, r, layer)
        out["d_x"] = g
        if c["gate"] != "none":
            dg = c["scale"] * g * u
            out["d_gate"] = {"channel": dg.sum((0, 1)), "sequence": dg.sum(1, keepdim=True), "token": dg}[c["gate"]]
        g = c["scale"] * gate * g
        if c["post"]:
            out["d_post_w"] = (g * b_unit).sum((0, 1))
            if layer:
                out["d_post_bias"] = g.sum((0, 1))
            g = _exact_unit_backward(g * (v["post_w"] + add), b_unit, b_r, layer)
        out["d_branch"] = g
    return out


def _exact_rotary(st):
    rot, turn = st["case"]["rot"], st["case"]["interleaved"]
    pair = torch.polar(torch.full_like(st["freq"], st["factor"]).expand(*st["positions"].shape, -1),
                       st["positions"].double().unsqueeze(-1) * st["freq"])[:, :, None]

    def turned(t, by):
        t = t.detach().double()
        z = t[..., :rot].unflatten(-1, (rot // 2, 2) if turn else (2, rot // 2))
        z = torch.complex(*(z.unbind(-1) if turn else z.unbind(-2))) * by
        t = t.clone()
        t[..., :rot] = torch.stack((z.real, z.imag), -1 if turn else -2).flatten(-2)
        return t

    out = {n: turned(st[n], pair) for n in ("q", "k")}
    if st["case"]["train"]:
        out.update({n: turned(st[n], pair.conj()) for n in ("dq", "dk")})
    return out
