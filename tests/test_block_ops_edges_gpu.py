"""Calls of the block operators at their edges: derivatives that they do not have, gradients that lie
oddly, batches without rows, results written in place, and column sums over many rows."""

import pytest
import torch

from test_residual_norm_gpu import BF, EPS, F32, HF, chain_of, close, forward64, inputs, unit_back

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------ derivatives
def forward_calls():
    """Each operator as a function of one tensor, for each of its differentiable arguments."""
    from saelens_b200 import ops

    st = ops.StatusWord("cuda")
    w, s = ops.quantize_fp8(torch.randn(128, 64, device="cuda"), 128)
    x, a, v = torch.randn(3, 64, device="cuda"), torch.randn(3, 64, device="cuda"), torch.randn(64, device="cuda")
    q, f = torch.randn(1, 3, 2, 64, device="cuda"), torch.ones(32, device="cuda", dtype=torch.float64)
    norm = {"x": x, "branch": a, "weight": v, "bias": v, "post_weight": v, "post_bias": v, "gate": v}
    calls = {"norm " + n: (lambda t, n=n: ops.residual_norm(**{**norm, n: t}, kind="layer"), norm[n]) for n in norm}
    calls["linear x"] = (lambda t: ops.linear_fp8(t, w, s, status=st), x)
    calls["linear x, own status"] = (lambda t: ops.linear_fp8(t, w, s), x)
    calls["linear bias"] = (lambda t: ops.linear_fp8(x, w, s, t, status=st), torch.zeros(128, device="cuda"))
    calls["linear scale"] = (lambda t: ops.linear_fp8(x, w, t, status=st), s)
    calls["rotary q"] = (lambda t: ops.rotary(t, q, f), q)
    calls["rotary k"] = (lambda t: ops.rotary(q, t, f), q)
    calls["rotary freq"] = (lambda t: ops.rotary(q, None, t), f)
    calls["rotary in place"] = (lambda t: ops.rotary(t, None, f, inplace=True), q.clone())
    return calls


CALLS = ["norm " + n for n in ("x", "branch", "weight", "bias", "post_weight", "post_bias", "gate")] + [
    "linear x", "linear x, own status", "linear bias", "linear scale", "rotary q", "rotary k", "rotary freq", "rotary in place"]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    """Forward-mode derivatives are not computed; a tangent may not be dropped without a word."""
    import torch.autograd.forward_ad as fw

    call, t = forward_calls()[name]
    with torch.set_grad_enabled(grad), fw.dual_level():
        call(t)
        with pytest.raises(ValueError, match="forward-mode"):
            call(fw.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("name", ["x", "branch", "weight", "bias", "post_weight", "post_bias", "gate"])
def test_the_gradient_of_the_norms_gradient_is_refused(name):
    """The first gradient depends on every input, whether or not the incoming gradient does."""
    from saelens_b200 import ops

    v = inputs(5, 64, F32, "layer", True, ())
    v[name].requires_grad_()
    s, y = ops.residual_norm(**v, kind="layer")
    (g,) = torch.autograd.grad(s.sum() + y.sum(), [v[name]], create_graph=True)
    (want,) = torch.autograd.grad(sum(t.sum() for t in ops.residual_norm(**v, kind="layer")), [v[name]])
    assert torch.equal(g.detach(), want)
    with pytest.raises(RuntimeError, match="once"):
        g.square().sum().backward()
    # a loss that does not go through the first gradient is not concerned
    s, y = ops.residual_norm(**v, kind="layer")
    (g,) = torch.autograd.grad(y.sum(), [v[name]], create_graph=True)
    (y.square().sum() + g.detach().sum()).backward()
    assert torch.isfinite(v[name].grad).all()


# ------------------------------------------------------------------------------------ odd layouts, no rows
@pytest.mark.parametrize("d", [8200, 16384])
@pytest.mark.parametrize("start,wide", [(0, 3), (3, 5), (8, 8)])
def test_wide_rows_whose_gradient_is_a_view(d, start, wide):
    """What concatenation and padding send back: a narrowed view whose rows start anywhere."""
    from saelens_b200 import ops

    v = {n: t.requires_grad_() for n, t in inputs(3, d, BF, "rms", True, None).items()}
    s, y = ops.residual_norm(**v, eps=EPS)
    gs, gy = (torch.randn(3, d + wide + 3, device="cuda").to(BF)[:, start : start + d] for _ in range(2))
    names = list(v.values())
    for outs, grads in (((s, y), (gs, gy)), ((s,), (gs,)), ((y,), (gy,))):
        got = torch.autograd.grad(outs, names, grads, retain_graph=True, allow_unused=True)
        want = torch.autograd.grad(outs, names, [g.contiguous() for g in grads], retain_graph=True, allow_unused=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("x,gate", [((2, 0), (2, 1)), ((2, 0), (2, 0)), ((0, 3), (0, 1)), ((0, 3), (0, 3)), ((0, 3), (1, 1)), ((2, 0), ()),
                                    ((2, 0, 3), (2, 1, 1)), ((2, 0, 3), (2, 0, 1)), ((2, 3, 0), (2, 3, 1))])
def test_gradients_of_a_gate_without_rows(x, gate):
    from saelens_b200 import ops

    v = {n: t.requires_grad_() for n, t in inputs(None, 64, F32, "rms", True, gate, x).items()}
    s, y = ops.residual_norm(**v)
    assert s.shape == y.shape == (*x, 64)
    got = torch.autograd.grad((s.sum() + y.sum()), list(v.values()))
    for name, g in zip(v, got):
        assert g.shape == v[name].shape and (g == 0).all(), name


# ------------------------------------------------------------------------------------ in place
def test_results_in_place_count_as_changes():
    """A tensor that autograd saved and that an operator then overwrites is noticed."""
    from saelens_b200 import ops

    f = torch.ones(32, device="cuda", dtype=torch.float64)
    w = torch.randn(64, device="cuda", requires_grad=True)
    for one in (lambda q, k: q, lambda q, k: k):
        q, k = torch.randn(1, 3, 2, 64, device="cuda"), torch.randn(1, 3, 2, 64, device="cuda")
        y = (one(q, k) * w).sum()
        ops.rotary(q, k, f, inplace=True)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()
    a, sa = ops.quantize_fp8(torch.randn(4, 64, device="cuda"), 1)
    b, sb = ops.quantize_fp8(torch.randn(64, 64, device="cuda"), 128)
    out = torch.randn(4, 64, device="cuda")
    y = (out * w).sum()
    ops.gemm_fp8(a, sa, b, sb, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():  # such tensors count nothing
        q = torch.randn(1, 3, 2, 64, device="cuda")
        want = ops.rotary(q, None, f)
        assert torch.equal(ops.rotary(q, None, f, inplace=True), want)
    assert torch.equal(ops.rotary(want.clone(), None, f, inplace=True), ops.rotary(want, None, f))
    ops.rotary(q, None, f, inplace=True)  # written outside as well, as before
    leaf = torch.zeros(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="out"):
        ops.gemm_fp8(a, sa, b, sb, out=leaf)
    with torch.no_grad():
        ops.gemm_fp8(a, sa, b, sb, out=leaf)


def test_rows_of_out_that_overlap_are_refused():
    from saelens_b200 import ops

    a, sa = ops.quantize_fp8(torch.randn(4, 64, device="cuda"), 1)
    b, sb = ops.quantize_fp8(torch.randn(96, 64, device="cuda"), 128)
    buf = torch.zeros(4 * 96, device="cuda")
    for out in (buf[:96].expand(4, 96), buf.as_strided((4, 96), (95, 1)), buf.as_strided((4, 96), (32, 1))):
        with pytest.raises(RuntimeError, match="rows apart"):
            ops.gemm_fp8(a, sa, b, sb, out=out)
    assert (buf == 0).all()
    want = ops.gemm_fp8(a, sa, b, sb, out_dtype=F32)
    assert torch.equal(ops.gemm_fp8(a, sa, b, sb, out=buf.view(4, 96)), want)
    one = buf[:96].expand(1, 96)
    assert torch.equal(ops.gemm_fp8(a[:1], sa[:1], b, sb, out=one), ops.gemm_fp8(a[:1], sa[:1], b, sb, out_dtype=F32))


# ------------------------------------------------------------------------------------ many rows
MANY = [
    # rows of 64: 15 groups a block, 2220 rows at once; sequences below, at and above a group's three rows
    (64, F32, "layer", True, (2500, 2)), (64, BF, "rms", True, (1681, 3)), (64, HF, "rms", False, (721, 7)), (64, F32, "rms", True, (5, 1009)),
    # 5 groups, 740 rows at once
    (768, F32, "layer", True, (8, 513)), (768, BF, "layer", True, (684, 6)), (768, F32, "rms", True, (1026, 4)), (760, F32, "rms", False, (500, 9)),
    # one group, sums in shared memory; sequences of a unit's rows, fewer and more
    (4096, BF, "rms", True, (3, 1001)), (4096, BF, "layer", True, (300, 10)), (4096, F32, "rms", False, (273, 11)), (2056, F32, "layer", True, (600, 5)),
    # single values, 256 and 512 threads
    (1001, BF, "layer", True, (3, 1003)), (1001, F32, "rms", True, (375, 8)), (3001, F32, "rms", True, (429, 7)), (3001, BF, "layer", False, (5, 600)),
]


@pytest.mark.parametrize("d,dtype,kind,post,lead", MANY)
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
def test_gradients_over_many_rows(d, dtype, kind, post, lead, gate):
    """Several rows a unit: sums carried from row to row, buffers that alternate, sequences that begin
    and end inside a unit, units that the last rows do not fill."""
    from saelens_b200 import ops

    layer, (b, s) = kind == "layer", lead
    shape = {None: None, "channel": (), "sequence": (b, 1), "token": (b, s)}[gate]
    v = {n: t.requires_grad_() for n, t in inputs(None, d, dtype, kind, post, shape, lead).items()}
    scale = 1.0 if gate is None else -0.75
    stream, normed = ops.residual_norm(**v, kind=kind, eps=EPS, scale=scale)
    ds, dn = (torch.randn(*lead, d, device="cuda").to(dtype) for _ in range(2))
    got = dict(zip(v, torch.autograd.grad((stream, normed), list(v.values()), (ds, dn))))
    r = forward64(v, kind, False, scale, stored=stream)
    f, dsd, dnd = r["f"], ds.double(), dn.double()
    rows = (0, 1)
    want, mags = {}, {}
    want["weight"], mags["weight"] = (dnd * r["unit"]).sum(rows), (dnd.abs() * r["t_mag"]).sum(rows)
    if layer:
        want["bias"], mags["bias"] = dnd.sum(rows), dnd.abs().sum(rows)
    pre, pre_mag = unit_back(dnd * r["w"], r["unit"], r["r"], layer)
    pre_mag = pre_mag + r["r"] * r["t_mag"] * (dnd * r["w"] * r["t_mag"]).abs().mean(-1, keepdim=True)
    g, g_mag = dsd + pre, dsd.abs() + pre_mag
    want["x"], mags["x"] = g, g_mag
    if post:
        b_mag = r["b_unit"].abs() + (r["b_r"] * f["branch"].abs().mean(-1, keepdim=True) if layer else 0)
    if gate is not None:
        # from the branch itself: under a gate of 0 (randn gives one in 10^7 values) nothing of it is left in
        # the stream's magnitude, while the gate's gradient is the rounded sums' product with it as ever
        u_mag = b_mag * f["post_weight"].abs() + f.get("post_bias", r["u"] * 0).abs() if post else f["branch"].abs()
        p, m = scale * g * r["u"], abs(scale) * g_mag * u_mag
        if gate != "token":
            p, m = (t.sum(rows if gate == "channel" else 1, keepdim=True) for t in (p, m))
        want["gate"], mags["gate"] = p.reshape(v["gate"].shape), m.reshape(v["gate"].shape)
    du, du_mag = r["g"] * g, r["g"].abs() * g_mag
    if post:
        want["post_weight"], mags["post_weight"] = (du * r["b_unit"]).sum(rows), (du_mag * b_mag).sum(rows)
        if layer:
            want["post_bias"], mags["post_bias"] = du.sum(rows), du_mag.sum(rows)
        h, h_mag = du * f["post_weight"], du_mag * f["post_weight"].abs()
        du, _ = unit_back(h, r["b_unit"], r["b_r"], layer)
        du_mag = r["b_r"] * (h_mag + b_mag * (h_mag * b_mag).mean(-1, keepdim=True) * 2 + h_mag.mean(-1, keepdim=True))
    want["branch"], mags["branch"] = du, du_mag
    assert set(got) == set(want)
    # a value's own roundings are those of the small cases; a column adds a unit's rows one by one (a
    # 148th of all or 11 at most), 15 groups, 16 parts of at most 8 x 148 blocks and the 16 parts, a
    # sequence that spans units one part for each
    chain = 3 * chain_of(d) + max(b * s // 148 + 8, 11) + 15 + 8 * 148 // 16 + 16
    for name in v:
        close(got[name], want[name], mags[name], chain + (s if name == "gate" else 0), name)
    again = torch.autograd.grad(ops.residual_norm(**v, kind=kind, eps=EPS, scale=scale), list(v.values()), (ds, dn))
    assert all(torch.equal(got[n], t) for n, t in zip(v, again))  # the same bits again
