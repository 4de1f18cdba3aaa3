"""Rotary positions against complex products in 64 bits.

Tolerance: the fraction of a turn is rounded to fp32 (2^-25 of at most half a turn, an angle of
2^-24 pi), the sine and cosine are off by a few units in the last place, scaled, multiplied and added:
16 2^-24 (|a| + |b|) factor covers them; the output is rounded once, by eps / 2.  Positions enter in
64 bits: p * freq / 2 pi is off by 2^-51 of itself, and so is the reference's angle."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def check(got, x, pos, freq, interleaved, factor=1.0, inverse=False):
    rot = 2 * freq.numel()
    x = x.detach()
    angle = (pos.double()[..., None] * freq)[:, :, None]
    c, s = torch.cos(angle) * factor, torch.sin(angle) * factor * (-1 if inverse else 1)
    f = x.double()
    a, b = (f[..., 0:rot:2], f[..., 1:rot:2]) if interleaved else (f[..., : rot // 2], f[..., rot // 2 : rot])
    na, nb = a * c - b * s, b * c + a * s
    far = (2.0**-50 * angle.abs() + 16 * 2.0**-24) * abs(factor) * (a.abs() + b.abs())
    ref, tol = f.clone(), torch.zeros_like(f)
    if interleaved:
        ref[..., 0:rot:2], ref[..., 1:rot:2] = na, nb
        tol[..., 0:rot:2] = tol[..., 1:rot:2] = far
    else:
        ref[..., : rot // 2], ref[..., rot // 2 : rot] = na, nb
        tol[..., : rot // 2] = tol[..., rot // 2 : rot] = far
    tol = tol + torch.finfo(got.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(got.dtype).smallest_normal
    assert got.shape == x.shape and got.dtype == x.dtype
    assert ((got.double() - ref).abs() <= tol).all()
    assert torch.equal(got[..., rot:], x[..., rot:])  # passed through


def freqs(rot, base=10000.0):
    from saelens_b200 import ops

    return ops.rotary_frequencies(rot, base, device="cuda")[0]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("b,s,h,kv,d,rot", [(1, 1, 1, 1, 2, 2), (2, 33, 8, 2, 128, 128), (3, 7, 5, 5, 64, 16), (2, 9, 4, 1, 80, 20),
                                            (1, 257, 3, 1, 34, 6), (64, 1, 32, 8, 128, 128), (2, 5, 2, 2, 256, 64),
                                            (1, 3, 1, 1, 8192, 8190), (2, 1500, 1, 1, 16, 8)])
def test_turns(b, s, h, kv, d, rot, dtype, interleaved):
    from saelens_b200 import ops

    q, k = (torch.randn(b, s, n, d, device="cuda").to(dtype) for n in (h, kv))
    pos = torch.randint(-50, 1_000_000, (b, s), device="cuda")
    f = freqs(rot)
    qo, ko = ops.rotary(q, k, f, positions=pos, interleaved=interleaved, factor=1.25)
    check(qo, q, pos, f, interleaved, 1.25)
    check(ko, k, pos, f, interleaved, 1.25)
    assert torch.equal(ops.rotary(q, None, f, positions=pos.int(), interleaved=interleaved, factor=1.25), qo)
    qi, ki = q.clone(), k.clone()
    back = ops.rotary(qi, ki, f, positions=pos, interleaved=interleaved, factor=1.25, inplace=True)
    assert back[0] is qi and torch.equal(qi, qo) and torch.equal(ki, ko)


def test_positions_and_strides():
    from saelens_b200 import ops

    b, s, h, kv, d = 3, 17, 4, 2, 64
    f = freqs(d)
    qkv = torch.randn(b, s, (h + 2 * kv) * d + 24, device="cuda").to(BF)
    q, k = qkv[..., 8 : 8 + h * d].view(b, s, h, d), qkv[..., 8 + h * d : 8 + (h + kv) * d].view(b, s, kv, d)
    base = torch.arange(s, device="cuda")
    want = ops.rotary(q.contiguous(), k.contiguous(), f)
    check(want[0], q, base.expand(b, s), f, False)
    for got in (ops.rotary(q, k, f), ops.rotary(q, k, f, positions=base), ops.rotary(q, k, f, positions=base.expand(b, s)),
                ops.rotary(q, k, f, positions=base[None].int())):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    far = ops.rotary(q, k, f, offset=1 << 20)
    check(far[0], q, base.expand(b, s) + (1 << 20), f, False)
    col = torch.tensor([[5], [9], [100]], device="cuda")
    check(ops.rotary(q, None, f, positions=col), q, col.expand(b, s), f, False)
    # another order of axes, odd offsets, and views turned in place beside what they leave alone
    t = torch.randn(b, h, s, d + 1, device="cuda")
    view = t.transpose(1, 2)[..., 1:]
    check(ops.rotary(view, None, f), view, base.expand(b, s), f, False)
    turned = torch.cat([x.reshape(b, s, -1) for x in ops.rotary(q, k, f)], -1)
    before = qkv.clone()
    ops.rotary(q, k, f, inplace=True)
    assert torch.equal(qkv[..., 8 : 8 + (h + kv) * d], turned)
    assert torch.equal(qkv[..., :8], before[..., :8]) and torch.equal(qkv[..., 8 + (h + kv) * d :], before[..., 8 + (h + kv) * d :])
    x = torch.randn(2, 3, 4, 128, device="cuda")[..., ::2]
    check(ops.rotary(x, None, f), x, torch.arange(3, device="cuda").expand(2, 3), f, False)
    assert ops.rotary(q[:, :0], k[:, :0], f)[1].shape == (b, 0, kv, d) and ops.rotary(q[:0], None, f).shape == (0, s, h, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rotary(view, None, f)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ops.rotary(view, None, f))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradients(dtype, interleaved):
    from saelens_b200 import ops

    q, k = (torch.randn(2, 11, n, 72, device="cuda").to(dtype).requires_grad_() for n in (6, 2))
    pos = torch.randint(0, 9000, (2, 11), device="cuda")
    f = freqs(24)
    qo, ko = ops.rotary(q, k, f, positions=pos, interleaved=interleaved, factor=0.5)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk), retain_graph=True)
    check_grad = lambda d, g: check(d, g, pos, f, interleaved, 0.5, inverse=True)  # noqa: E731
    # channels that pass through have the gradient itself: `check` compares them bit for bit
    check_grad(dq, gq)
    check_grad(dk, gk)
    (only,) = torch.autograd.grad(ko, k, gk, retain_graph=True)
    assert torch.equal(only, dk)
    (only,) = torch.autograd.grad(qo.sum(), q, retain_graph=True)  # an expanded gradient
    check_grad(only, torch.ones_like(q))
    if dtype == F32:
        # differences: the map is linear, so a unit step is exact up to rounding
        v = torch.randn_like(q)
        step = ops.rotary(q.detach() + v, None, f, positions=pos, interleaved=interleaved, factor=0.5) - qo.detach()
        lhs, rhs = (step.double() * gq.double()).sum(), (dq.double() * v.double()).sum()
        assert (lhs - rhs).abs() <= 64 * 2.0**-24 * ((q.detach().abs() + v.abs()).sum() * gq.abs().max())
        # the gradient of the gradient is the rotation again
        gq2 = gq.clone().requires_grad_()
        (d1,) = torch.autograd.grad(qo, q, gq2, create_graph=True)
        (d2,) = torch.autograd.grad(d1, gq2, v)
        check(d2, v, pos, f, interleaved, 0.5)


def test_scaled_contexts_turn_by_their_frequencies():
    from saelens_b200 import ops

    q = torch.randn(1, 40, 2, 128, device="cuda")
    for scaling in ({"rope_type": "linear", "factor": 4.0}, {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192},
                    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
                    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}):
        f, factor = ops.rotary_frequencies(128, 500000.0, scaling, n_positions=100_000, device="cuda")
        check(ops.rotary(q, None, f, offset=99_000, factor=factor), q, torch.arange(99_000, 99_040, device="cuda")[None], f, False, factor)


def test_captured_graph_reads_new_positions():
    from saelens_b200 import ops

    q, k = torch.randn(8, 1, 4, 64, device="cuda").to(BF), torch.randn(8, 1, 2, 64, device="cuda").to(BF)
    pos = torch.zeros(8, 1, dtype=torch.int64, device="cuda")
    f = freqs(64)
    ops.rotary(q, k, f, positions=pos)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.rotary(q, k, f, positions=pos)
    for p in (3, 70_000):
        pos.fill_(p)
        g.replay()
        want = ops.rotary(q, k, f, positions=pos)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        check(out[0], q, pos, f, False)


def test_beyond_32_bit_offsets():
    from saelens_b200 import ops

    s = 525_001
    q = torch.empty(1, s, 32, 128, device="cuda", dtype=BF).normal_()  # 2.15e9 values
    f = freqs(128)
    out = ops.rotary(q, None, f)
    for a, b in ((0, 3), (s - 3, s)):
        check(out[:, a:b], q[:, a:b], torch.arange(a, b, device="cuda")[None], f, False)


def test_in_place_on_views_of_one_tensor():
    """q and k may interleave head by head, but not hold a value in common."""
    from saelens_b200 import ops

    f = freqs(64)
    pairs = torch.randn(2, 5, 4, 2, 64, device="cuda")
    q, k = pairs[..., 0, :], pairs[..., 1, :]
    want = ops.rotary(q, k, f)
    ops.rotary(q, k, f, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    halves = torch.randn(2, 10, 4, 64, device="cuda")
    q, k = halves[:, :5], halves[:, 5:]
    want = ops.rotary(q, k, f)
    ops.rotary(q, k, f, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    x = torch.randn(2, 5, 4, 64, device="cuda")
    for q, k in ((x, x), (x[:, :, :3], x[:, :, 1:]), (x, x[:, :, 3:]), (x[:, :4], x[:, 1:]), (x[..., :34], x[..., 30:])):
        with pytest.raises(ValueError, match="share"):
            ops.rotary(q, k, freqs(32), inplace=True)
    ops.rotary(x[:, :, :3], x[:, :, 3:], f, inplace=True)


def test_refusals_on_the_device():
    from saelens_b200 import ops

    q = torch.randn(2, 3, 4, 64, device="cuda")
    f = freqs(64)
    for bad in (lambda: ops.rotary(q, None, f.float()), lambda: ops.rotary(q, None, torch.cat([f, f])), lambda: ops.rotary(q, None, f.cpu()),
                lambda: ops.rotary(q.double(), None, f), lambda: ops.rotary(q[0], None, f), lambda: ops.rotary(q, q[:1], f),
                lambda: ops.rotary(q, q.to(BF), f), lambda: ops.rotary(q, q.cpu(), f),
                lambda: ops.rotary(q, None, f, positions=torch.zeros(2, 2, dtype=torch.int64, device="cuda")),
                lambda: ops.rotary(q, None, f, positions=torch.zeros(2, 3, device="cuda")),
                lambda: ops.rotary(q, None, f, positions=torch.zeros(2, 3, dtype=torch.int64)),
                lambda: ops.rotary(q, None, f, positions=torch.zeros(2, 3, dtype=torch.int64, device="cuda"), offset=2),
                lambda: ops.rotary(q[:1].expand(2, -1, -1, -1), None, f, inplace=True),
                lambda: ops.rotary(q.clone().requires_grad_(), None, f, inplace=True),
                lambda: ops.rotary(torch.randn(1, 2, 2, 128, device="cuda")[..., ::2], None, f, inplace=True)):
        with pytest.raises(ValueError):
            bad()
