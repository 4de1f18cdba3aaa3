"""The residual update between two norms against its definition in 64 bits.

Tolerances.  A fp32 operation is off by 2^-24 of its value; a sum of n addends in the kernel's order
by at most (its longest chain + 1) 2^-24 of the sum of absolute values; an output is rounded once, by
eps / 2.  The normed rows are checked against the norm of the stream that came back (the definition
reads the stored stream), so no rounding of the stream enters twice."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24
EPS = 1e-6


def unit(t, layer):
    if layer:
        t = t - t.mean(-1, keepdim=True)
    r = (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return t * r, r


def inputs(rows, d, dtype, kind, post, gate, lead=None):
    lead = lead or (rows,)
    v = {"x": torch.randn(*lead, d, device="cuda") * 2 + 0.3, "branch": torch.randn(*lead, d, device="cuda") - 0.2,
         "weight": torch.randn(d, device="cuda")}
    if kind == "layer":
        v["bias"] = torch.randn(d, device="cuda")
    if post:
        v["post_weight"] = torch.randn(d, device="cuda")
        if kind == "layer":
            v["post_bias"] = torch.randn(d, device="cuda")
    if gate is not None:
        v["gate"] = torch.randn(*gate, d, device="cuda")
    return {n: t.to(dtype) for n, t in v.items()}


def forward64(v, kind, one_plus, scale, stored=None):
    """Stream, normed (of `stored`) and what the gradients need, with the tolerances' magnitudes."""
    layer, add = kind == "layer", 1.0 if one_plus else 0.0
    f = {n: t.detach().double() for n, t in v.items()}
    u, mu = f["branch"], f["branch"].abs()
    b_unit = b_r = None
    if "post_weight" in f:
        b_unit, b_r = unit(u, layer)
        pw = f["post_weight"] + add
        u = b_unit * pw + f.get("post_bias", 0.0)
        mu = (b_unit.abs() + (b_r * f["branch"].abs().mean(-1, keepdim=True) if layer else 0)) * pw.abs() + f.get("post_bias", u * 0).abs()
    g = scale * f["gate"] if "gate" in f else torch.full((), scale, dtype=torch.float64, device="cuda")
    stream = f["x"] + g * u
    t, r = unit(stream if stored is None else stored.double(), layer)
    w = f["weight"] + add
    normed = t * w + f.get("bias", 0.0)
    t_mag = t.abs() + (r * stream.abs().mean(-1, keepdim=True) if layer else 0)
    return {"stream": stream, "normed": normed, "unit": t, "r": r, "w": w, "u": u, "b_unit": b_unit, "b_r": b_r, "g": g,
            "stream_mag": f["x"].abs() + g.abs() * mu, "t_mag": t_mag, "normed_mag": t_mag * w.abs() + f.get("bias", t * 0).abs(), "f": f}


def close(got, ref, mag, chain, name):
    eps = torch.finfo(got.dtype).eps / 2
    tol = (chain + 24) * U * mag
    tol = tol + eps * (ref.abs() + tol) + torch.finfo(got.dtype).smallest_normal
    worst = ((got.double() - ref).abs() - tol).max().item()
    assert not torch.isnan(got).any() and worst <= 0, (name, worst)


def chain_of(d):  # a thread's values, the butterfly, the warps; twice for a mean and a variance
    return 2 * (-(-d // 256) * 8 + 5 + 8)


CASES = [(1, 4096, BF, "rms", False, False), (3, 8, BF, "rms", True, True), (77, 768, F32, "layer", True, False),
         (5, 3584, BF, "rms", True, True), (9, 1, F32, "layer", True, False), (130, 7, HF, "rms", False, True),
         (33, 1000, HF, "layer", False, False), (4, 2049, BF, "layer", True, True), (2, 8191, F32, "rms", True, False),
         (3, 16384, BF, "layer", True, False), (2, 8200, F32, "rms", True, True), (600, 64, BF, "layer", True, False)]


@pytest.mark.parametrize("rows,d,dtype,kind,post,one_plus", CASES)
@pytest.mark.parametrize("gate", [None, "channel", "token"])
def test_forward(rows, d, dtype, kind, post, one_plus, gate):
    from saelens_b200 import ops

    v = inputs(rows, d, dtype, kind, post, {"channel": (), "token": (rows,)}.get(gate))
    scale = 0.625 if gate else 1.0
    stream, normed = ops.residual_norm(**v, kind=kind, eps=EPS, one_plus=one_plus, scale=scale)
    assert stream.dtype == dtype and stream.shape == v["x"].shape and normed.shape == stream.shape
    ref = forward64(v, kind, one_plus, scale, stored=stream)
    close(stream, ref["stream"], ref["stream_mag"], chain_of(d), "stream")
    close(normed, ref["normed"], ref["normed_mag"], chain_of(d), "normed")
    again = ops.residual_norm(**v, kind=kind, eps=EPS, one_plus=one_plus, scale=scale)
    assert torch.equal(again[0], stream) and torch.equal(again[1], normed)


def unit_back(g, t, r, layer):
    out = g - t * (g * t).mean(-1, keepdim=True)
    mag = g.abs() + t.abs() * (g * t).abs().mean(-1, keepdim=True)
    if layer:
        out, mag = out - g.mean(-1, keepdim=True), mag + g.abs().mean(-1, keepdim=True)
    return out * r, mag * r


LEAD = (3, 7, 5)


@pytest.mark.parametrize("d,dtype,kind,post,one_plus", [(64, F32, "rms", False, False), (768, F32, "layer", True, False),
                                                       (512, BF, "rms", True, True), (129, HF, "layer", True, False),
                                                       (4096, BF, "layer", True, True), (2500, F32, "rms", True, True),
                                                       (1, F32, "rms", True, False), (6152, F32, "layer", True, False)])
@pytest.mark.parametrize("gate", [None, (), (3, 1, 1), (3, 7, 1), LEAD])
@pytest.mark.parametrize("which", ["both", "stream", "normed"])
def test_gradients(d, dtype, kind, post, one_plus, gate, which):
    from saelens_b200 import ops

    layer = kind == "layer"
    v = {n: t.requires_grad_() for n, t in inputs(None, d, dtype, kind, post, gate, LEAD).items()}
    scale = 1.0 if gate is None else -0.75
    stream, normed = ops.residual_norm(**v, kind=kind, eps=EPS, one_plus=one_plus, scale=scale)
    ds, dn = (torch.randn(*LEAD, d, device="cuda").to(dtype) for _ in range(2))
    if which == "both":
        got = torch.autograd.grad((stream, normed), list(v.values()), (ds, dn), allow_unused=True)
    elif which == "stream":
        got, dn = torch.autograd.grad(stream, list(v.values()), ds, allow_unused=True), dn * 0
    else:
        got, ds = torch.autograd.grad(normed, list(v.values()), dn, allow_unused=True), ds * 0
    got = dict(zip(v, got))
    r = forward64(v, kind, one_plus, scale, stored=stream)
    dsd, dnd = ds.double(), dn.double()
    n = 105
    rows = (0, 1, 2)
    chain = chain_of(d)
    # the unit rows themselves are off by chain U t_mag; their products carry that on
    want, mags = {}, {}
    want["weight"], mags["weight"] = (dnd * r["unit"]).sum(rows), (dnd.abs() * r["t_mag"]).sum(rows) * (1 + n / 8)
    if layer:
        want["bias"], mags["bias"] = dnd.sum(rows), dnd.abs().sum(rows) * (1 + n / 8)
    pre, pre_mag = unit_back(dnd * r["w"], r["unit"], r["r"], layer)
    pre_mag = pre_mag + r["r"] * r["t_mag"] * (dnd * r["w"] * r["t_mag"]).abs().mean(-1, keepdim=True)
    g = dsd + pre
    g_mag = dsd.abs() + pre_mag
    want["x"], mags["x"] = g, g_mag
    if gate is not None:
        dims = [i for i in rows if ((1,) * (3 - len(gate)) + tuple(gate))[i] == 1]
        u_mag = r["stream_mag"] - r["f"]["x"].abs()
        u_mag = u_mag / r["g"].abs().clamp_min(1e-30)
        p, m = scale * g * r["u"], abs(scale) * g_mag * u_mag
        for i in dims:
            p, m = p.sum(i, keepdim=True), m.sum(i, keepdim=True)
        want["gate"], mags["gate"] = p.reshape(v["gate"].shape), m.reshape(v["gate"].shape) * (1 + n / 8)
    du, du_mag = r["g"] * g, r["g"].abs() * g_mag
    if post:
        pw = r["f"]["post_weight"] + (1.0 if one_plus else 0.0)
        b_mag = r["b_unit"].abs() + (r["b_r"] * r["f"]["branch"].abs().mean(-1, keepdim=True) if layer else 0)
        want["post_weight"], mags["post_weight"] = (du * r["b_unit"]).sum(rows), (du_mag * b_mag).sum(rows) * (1 + n / 8)
        if layer:
            want["post_bias"], mags["post_bias"] = du.sum(rows), du_mag.sum(rows) * (1 + n / 8)
        h, h_mag = du * pw, du_mag * pw.abs()
        du, _ = unit_back(h, r["b_unit"], r["b_r"], layer)
        du_mag = r["b_r"] * (h_mag + b_mag * (h_mag * b_mag).mean(-1, keepdim=True) * 2 + h_mag.mean(-1, keepdim=True))
    want["branch"], mags["branch"] = du, du_mag
    for name in v:
        if got[name] is None:
            raise AssertionError(f"no gradient of {name}")
        close(got[name], want[name], mags[name], 3 * chain, name)


def test_gradients_against_differences():
    """Central differences of the kernel's own fp32 forward: off by the rounding of two forwards over
    the step, and the step's third-order term."""
    from saelens_b200 import ops

    v = inputs(None, 96, F32, "layer", True, (3, 1, 1), LEAD)
    v = {n: t.requires_grad_() for n, t in v.items()}
    c = [torch.randn(*LEAD, 96, device="cuda") for _ in range(2)]

    def value(w):
        s, y = ops.residual_norm(**w, kind="layer", eps=EPS, scale=0.5)
        return (s.double() * c[0]).sum() + (y.double() * c[1]).sum()

    grads = dict(zip(v, torch.autograd.grad(value(v), list(v.values()))))
    for name in v:
        way = torch.randn_like(v[name])
        way /= way.norm()
        h = 2.0**-6
        moved = [value({**{n: t.detach() for n, t in v.items()}, name: v[name].detach() + s * h * way}) for s in (1, -1)]
        slope = ((moved[0] - moved[1]) / (2 * h)).item()
        want = (grads[name].double() * way).sum().item()
        # 105 * 96 outputs of size ~4 weighted ~1: rounding 2^-24 * 4 * sqrt(n) * a few over h, and h^2 terms
        assert abs(slope - want) <= 2e-2 + 2e-3 * abs(want), (name, slope, want)


def test_only_what_is_asked_for():
    from saelens_b200 import ops

    v = inputs(64, 256, BF, "rms", True, (64,))
    full = {n: t.clone().requires_grad_() for n, t in v.items()}
    s, y = ops.residual_norm(**full, eps=EPS)
    want = dict(zip(full, torch.autograd.grad(s.float().sum() + y.float().square().sum(), list(full.values()))))
    for name in v:
        w = {n: t.clone().requires_grad_(n == name) for n, t in v.items()}
        s, y = ops.residual_norm(**w, eps=EPS)
        (g,) = torch.autograd.grad(s.float().sum() + y.float().square().sum(), [w[name]])
        assert torch.equal(g, want[name]), name


def test_same_bits_as_the_single_norms():
    """With `round_branch`, what the producer computes norm by norm."""
    from saelens_b200 import ops
    from saelens_b200.ops import native

    for d in (64, 768, 3584, 4096, 16384):
        x, a = (torch.randn(37, d, device="cuda").to(BF) for _ in range(2))
        w, p, b, pb = (torch.randn(d, device="cuda").to(BF) for _ in range(4))
        s, y = ops.residual_norm(x, a, w, eps=EPS, one_plus=True, post_weight=p, round_branch=True)
        want = x + native().rmsnorm(a, p, EPS, True)
        assert torch.equal(s, want) and torch.equal(y, native().rmsnorm(want, w, EPS, True)), d
        s, y = ops.residual_norm(x, a, w, b, eps=EPS, kind="layer", post_weight=p, post_bias=pb, round_branch=True)
        want = x + native().layernorm(a, p, pb, EPS)
        assert torch.equal(s, want) and torch.equal(y, native().layernorm(want, w, b, EPS)), d
        s, y = ops.residual_norm(x, a, w, eps=EPS)
        assert torch.equal(s, x + a) and torch.equal(y, native().rmsnorm(x + a, w, EPS, False)), d


def test_strides_streams_and_empty_rows():
    from saelens_b200 import ops

    wide = torch.randn(6, 20, 520, device="cuda").to(BF)
    w = torch.randn(256, device="cuda").to(BF)
    for x, a in ((wide[..., :256], wide[..., 264:]), (wide[..., 1:257], wide[..., 3:259]), (wide[:, ::2, :256], wide[:, 1::2, 8:264]),
                 (wide[:, :, ::2][..., :256], wide[:1, :, :256].expand(6, -1, -1))):
        got, want = ops.residual_norm(x, a, w, eps=EPS), ops.residual_norm(x.contiguous(), a.contiguous(), w, eps=EPS)
        assert torch.equal(got[0], want[0]) and torch.allclose(got[1].float(), want[1].float(), rtol=2.0**-7, atol=0)
    s, y = ops.residual_norm(wide[:0, :, :256], wide[:0, :, :256], w)
    assert s.shape == (0, 20, 256) and y.shape == s.shape
    x = wide[:0, :, :256].detach().requires_grad_()
    wl = w.clone().requires_grad_()
    s, y = ops.residual_norm(x, wide[:0, :, :256], wl)
    gx, gw = torch.autograd.grad((s.sum() + y.sum()), (x, wl))
    assert gx.shape == x.shape and (gw == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.residual_norm(wide[..., :256], wide[..., 264:], w, eps=EPS)
    torch.cuda.current_stream().wait_stream(side)
    want = ops.residual_norm(wide[..., :256], wide[..., 264:], w, eps=EPS)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_special_rows():
    """Rows of zeros give zeros, NaN and infinity stay in their rows."""
    from saelens_b200 import ops

    x, a = torch.randn(5, 64, device="cuda"), torch.randn(5, 64, device="cuda")
    w = torch.randn(64, device="cuda")
    x[1], a[1] = 0, 0
    want = ops.residual_norm(x, a, w, post_weight=w)
    assert (want[0][1] == 0).all() and (want[1][1] == 0).all()
    x[2, 3], a[4, 5] = float("nan"), float("inf")
    got = ops.residual_norm(x, a, w, post_weight=w)
    assert torch.equal(got[1][[0, 1, 3]], want[1][[0, 1, 3]]) and torch.isnan(got[1][2]).all() and torch.isnan(got[0][4]).any()


def test_captured_training_step():
    from saelens_b200 import ops

    v = {n: t.requires_grad_() for n, t in inputs(50, 512, BF, "layer", True, ()).items()}
    c = torch.randn(50, 512, device="cuda").to(BF)

    def step():
        s, y = ops.residual_norm(**v, kind="layer")
        return torch.autograd.grad((s, y), list(v.values()), (c, c))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        with torch.no_grad():
            for t in v.values():
                t.copy_(torch.randn_like(t))
        graph.replay()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_rows_beyond_32_bit_offsets():
    from saelens_b200 import ops

    rows, d = 525_001, 4096  # 2.15e9 values
    x = torch.empty(rows, d, device="cuda", dtype=BF).normal_()
    w = torch.randn(d, device="cuda").to(BF)
    s, y = ops.residual_norm(x, x, w, eps=EPS)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        a, b = ops.residual_norm(x[part].clone(), x[part].clone(), w, eps=EPS)
        assert torch.equal(s[part], a) and torch.equal(y[part], b)


def test_refusals_on_the_device():
    from saelens_b200 import ops

    x, w = torch.randn(2, 3, 64, device="cuda"), torch.randn(64, device="cuda")
    for kw in ({"branch": x[:1]}, {"branch": x.to(BF)}, {"weight": w[:63]}, {"weight": w.cpu()}, {"bias": w}, {"kind": "batch"},
               {"kind": "layer", "post_bias": w}, {"gate": x[:1]}, {"gate": x[..., :1]}, {"gate": x.cpu()}, {"x": x.double()},
               {"x": torch.zeros(2, 16392, device="cuda"), "branch": torch.zeros(2, 16392, device="cuda"), "weight": torch.zeros(16392, device="cuda")},
               {"x": torch.zeros(2, 8193, device="cuda"), "branch": torch.zeros(2, 8193, device="cuda"), "weight": torch.zeros(8193, device="cuda")}):
        with pytest.raises((ValueError, RuntimeError)):
            ops.residual_norm(**{"x": x, "branch": x, "weight": w, **kw})
    d = 16384  # four column sums of which do not fit, three do
    a = torch.randn(2, d, device="cuda").requires_grad_()
    v = [torch.randn(d, device="cuda").requires_grad_() for _ in range(4)]
    with pytest.raises(ValueError, match="do not fit"):
        ops.residual_norm(a, a.detach(), v[0], v[1], kind="layer", post_weight=v[2], post_bias=v[3])
    s, y = ops.residual_norm(a, a.detach(), v[0], v[1], kind="layer", post_weight=v[2])
    g = torch.ones_like(y).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y, a, g, create_graph=True)
