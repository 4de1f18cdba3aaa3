"""The 8-bit projections against the definition in 64 bits.

Tolerances.  Products of two e4m3 values are exact in fp32; a block's sum of 128 of them and the sum
over the blocks are fp32 sums, off by at most 2^-23 (a truncating adder's unit) times the number of
addends times the sum of the absolute terms; scaling rounds three times; the output is rounded once,
by eps / 2 of its value."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
LEAST = 448.0 * torch.finfo(F32).tiny


def quantize_ref(x, rows):
    """e4m3 values (as fp32) and scales, by torch operations in fp32."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // 128)
    t = torch.nn.functional.pad(x.float(), (0, kb * 128 - k, 0, mb * rows - m)).view(mb, rows, kb, 128)
    most = t.abs().amax(dim=(1, 3), keepdim=True).clamp_min(LEAST)
    q = (t * 0.4375 / most * 1024.0).to(torch.float8_e4m3fn).float()
    # by a tensor: torch divides by a number as a product with its rounded reciprocal
    return q.view(mb * rows, kb * 128)[:m, :k], (most / torch.full_like(most, 448.0))[:, 0, :, 0]


def spread(s, rows, m, k):
    return s.double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def weight(n, k, dtype=BF):
    from saelens_b200 import ops

    w = torch.randn(n, k, device="cuda")
    w[:, ::13] *= 3
    return ops.quantize_fp8(w.to(dtype), 128)


def product_ref(xq, xs, wq, ws, bias, transposed=False):
    """The product in 64 bits, and the same with absolute values."""
    n, k = wq.shape
    w = wq.double() * spread(ws, 128, n, k)
    w = w if transposed else w.T
    x = xq.double() * spread(xs, 1, *xq.shape)
    y = x @ w
    return (y if bias is None else y + bias.double()), x.abs() @ w.abs()


def check_product(y, ref, mag, reduction, bias=None):
    tol = (128 + -(-reduction // 128) + 8) * 2.0**-23 * (mag + (0 if bias is None else bias.abs().double()))
    tol = tol + torch.finfo(y.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal
    bad = (y.double() - ref).abs() - tol
    assert not torch.isnan(y).any() and bad.max() <= 0, (bad.max().item(), y.shape)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 129), (130, 257), (77, 1000), (200, 4096), (2500, 2048)])
def test_quantize_bits(m, k, dtype, rows):
    from saelens_b200 import ops

    x = torch.randn(m, k, device="cuda") * torch.logspace(-6, 4, m, device="cuda")[:, None]
    x = x.to(dtype)
    x[0, : min(k, 5)] = 0
    q, s = ops.quantize_fp8(x, rows)
    rq, rs = quantize_ref(x, rows)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and q.stride(0) % 16 == 0
    assert torch.equal(s, rs) and torch.equal(q.float(), rq)


def test_quantize_strided_and_special_values():
    from saelens_b200 import ops

    wide = torch.randn(40, 700, device="cuda").to(BF)
    for x in (wide[:, 3:300], wide[::2, 8:264], wide.T, wide[:, ::2]):
        q, s = ops.quantize_fp8(x, 1)
        rq, rs = quantize_ref(x, 1)
        assert torch.equal(s, rs) and torch.equal(q.float(), rq)
    x = torch.zeros(4, 256, device="cuda", dtype=F32)
    x[1, 3], x[2, 5], x[3, 7] = float("inf"), float("nan"), 1e-44
    q, s = ops.quantize_fp8(x, 1)
    assert (q[0].float() == 0).all() and s[0, 0] == torch.finfo(F32).tiny
    assert torch.isinf(s[1, 0]) and torch.isnan(q[1, 3].float()) and torch.isnan(s[2, 0]) and s[1, 1] == s[0, 0]
    assert torch.equal(torch.nan_to_num(q.float()), torch.nan_to_num(quantize_ref(x, 1)[0]))
    big = torch.full((1, 128), torch.finfo(BF).max, device="cuda", dtype=BF)
    q, s = ops.quantize_fp8(big, 1)
    assert (q.float() == 448).all() and torch.isfinite(s).all()
    assert ops.quantize_fp8(x[:0], 1)[1].shape == (0, 2)


SIZES = [(1, 128, 128), (1, 4096, 640), (1, 28672, 20000), (2, 14336, 8192), (2, 1, 1), (4, 9000, 6150), (5, 130, 129), (16, 1024, 257), (17, 1024, 384), (24, 3584, 520),
         (32, 333, 100), (33, 2048, 1000), (64, 640, 2048), (65, 640, 2048), (127, 100, 300), (129, 1152, 130),
         (333, 5120, 1111), (1000, 2056, 2304), (2048, 512, 6200),
         (333, 640, 7168), (300, 200, 30000)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype,with_bias", [(BF, True), (HF, False), (F32, True)])
def test_linear(m, k, n, dtype, with_bias):
    from saelens_b200 import ops

    wq, ws = weight(n, k)
    x = torch.randn(m, k, device="cuda").to(dtype)
    bias = torch.randn(n, device="cuda") if with_bias else None
    y = ops.linear_fp8(x, wq, ws, bias)
    assert y.shape == (m, n) and y.dtype == dtype and y.is_contiguous()
    xq, xs = quantize_ref(x, 1)
    check_product(y, *product_ref(xq, xs, wq, ws, bias), k, bias)
    assert torch.equal(y, ops.linear_fp8(x, wq, ws, bias))  # the same bits again


@pytest.mark.parametrize("m,k,n", SIZES)
def test_gemm_of_quantized_rows(m, k, n):
    from saelens_b200 import ops

    wq, ws = weight(n, k)
    xq, xs = ops.quantize_fp8(torch.randn(m, k, device="cuda").to(BF), 1)
    ref, mag = product_ref(xq.float(), xs, wq, ws, None)
    for dtype in (BF, HF, F32):
        check_product(ops.gemm_fp8(xq, xs, wq, ws, out_dtype=dtype), ref, mag, k)
    # into a slice of a wider, oddly strided buffer: nothing beside it changes
    buf = torch.full((m + 1, n + 5), 7.0, device="cuda", dtype=BF)
    check_product(ops.gemm_fp8(xq, xs, wq, ws, out=buf[:m, 2 : n + 2]), ref, mag, k)
    assert (buf[m] == 7).all() and (buf[:, :2] == 7).all() and (buf[:, n + 2 :] == 7).all()


@pytest.mark.parametrize("m,k,n", [(1, 128, 128), (1, 4096, 640), (3, 130, 129), (16, 256, 1024), (20, 1000, 384),
                                   (64, 640, 2048), (127, 100, 300), (333, 1111, 5120), (1030, 2304, 2056),
                                   (2000, 4100, 384)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_gradient_of_rows(m, k, n, dtype):
    from saelens_b200 import ops

    wq, ws = weight(n, k)
    x = torch.randn(m, k, device="cuda").to(dtype).requires_grad_()
    y = ops.linear_fp8(x, wq, ws)
    g = torch.randn(m, n, device="cuda").to(dtype)
    (dx,) = torch.autograd.grad(y, x, g, retain_graph=True)
    gq, gs = quantize_ref(g, 1)
    ref, mag = product_ref(gq, gs, wq, ws, None, transposed=True)
    check_product(dx, ref, mag, n)
    # against differences of the exact product along a direction: they differ by the quantisation of
    # g, at most 2^-4 of a value or half of the least step, 2^-10 scales
    v = torch.randn(m, k, device="cuda", dtype=torch.float64)
    w = wq.double() * spread(ws, 128, n, k)
    step = ((x.detach().double() + 0.5 * v) @ w.T - (x.detach().double() - 0.5 * v) @ w.T)
    err = 2.0**-4 * g.abs().double() + 2.0**-10 * spread(gs, 1, m, n)
    tol = ((err @ w.abs()) * v.abs()).sum() + (mag * v.abs()).sum() * 2.0**-7
    assert (step * g.double()).sum().sub((dx.double() * v).sum()).abs() <= tol
    # a gradient that is expanded or strided
    (e,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    one, _ = product_ref(*quantize_ref(torch.ones_like(g), 1), wq, ws, None, transposed=True)
    assert (e.double() - one).abs().max() <= 2.0**-6 * one.abs().max() + 1e-3


def test_shapes_streams_and_strides():
    from saelens_b200 import ops

    wq, ws = weight(300, 264)
    x = torch.randn(2, 3, 5, 264, device="cuda").to(BF)
    flat = ops.linear_fp8(x.reshape(-1, 264), wq, ws)
    assert torch.equal(ops.linear_fp8(x, wq, ws).reshape(-1, 300), flat)
    assert ops.linear_fp8(x[0, 0, 0], wq, ws).shape == (300,)
    assert ops.linear_fp8(x[:0], wq, ws).shape == (0, 3, 5, 300)
    wide = torch.randn(30, 1000, device="cuda").to(BF)
    for part in (wide[:, 7:271], wide[::3, 8:272], wide[:, :528:2], wide[:1].expand(30, -1)[:, :264]):
        assert torch.equal(ops.linear_fp8(part, wq, ws), ops.linear_fp8(part.contiguous(), wq, ws))
    # scales in another layout, a weight that is a row range of a larger one
    assert torch.equal(ops.linear_fp8(x, wq, ws.T.contiguous().T), ops.linear_fp8(x, wq, ws))
    assert torch.equal(ops.linear_fp8(x, wq[128:256], ws[1:2]), ops.linear_fp8(x, wq, ws)[..., 128:256])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.linear_fp8(x, wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y.reshape(-1, 300), flat)


@pytest.mark.parametrize("m", [1, 40, 200])
def test_from_a_new_thread(m):
    """A thread that has called nothing of CUDA before."""
    import threading

    from saelens_b200 import ops

    wq, ws = weight(300, 264)
    x = torch.randn(m, 264, device="cuda").to(BF)
    st = ops.StatusWord("cuda")
    torch.cuda.synchronize()
    got = []
    t = threading.Thread(target=lambda: got.append(ops.linear_fp8(x, wq, ws, status=st)))
    t.start()
    t.join()
    assert torch.equal(got[0], ops.linear_fp8(x, wq, ws, status=st))


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_a_bad_row_stays_alone(m):
    from saelens_b200 import ops

    wq, ws = weight(260, 384)
    x = torch.randn(m, 384, device="cuda").to(BF)
    want = ops.linear_fp8(x, wq, ws)
    x[0, 130], x[m // 2, 3] = float("nan"), float("inf")
    y = ops.linear_fp8(x, wq, ws)
    rows = sorted({0, m // 2})
    assert torch.isnan(y[rows]).all()
    keep = [i for i in range(m) if i not in rows]
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("m", [1, 24, 300])
def test_captured_graphs(m):
    """Two graphs of the same call, replayed in turn on changed inputs."""
    from saelens_b200 import ops

    wq, ws = weight(384, 640)
    st = ops.StatusWord("cuda")
    xs = [torch.randn(m, 640, device="cuda").to(BF) for _ in range(2)]
    for x in xs:
        ops.linear_fp8(x, wq, ws, status=st)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.linear_fp8(x, wq, ws, status=st))
        graphs.append(g)
    for _ in range(3):
        new = [torch.randn_like(x) for x in xs]
        for x, t in zip(xs, new):
            x.copy_(t)
        for g in graphs:
            g.replay()
        for t, o in zip(new, outs):
            assert torch.equal(o, ops.linear_fp8(t, wq, ws, status=st))
    st.check()


def test_outputs_beyond_32_bit_offsets():
    from saelens_b200 import ops

    m, n, k = 70001, 32768, 128
    wq, ws = weight(n, k)
    x = torch.randn(m, k, device="cuda").to(BF)
    y = ops.linear_fp8(x, wq, ws)
    for rows in (slice(0, 3), slice(65534, 65538), slice(m - 3, m)):
        xq, xs = quantize_ref(x[rows], 1)
        check_product(y[rows], *product_ref(xq, xs, wq, ws, None), k)


def test_refusals_on_the_device():
    from saelens_b200 import ops

    st = ops.StatusWord("cuda")
    wq, ws = weight(256, 256)
    x = torch.randn(4, 256, device="cuda").to(BF)
    xq, xs = ops.quantize_fp8(x, 1)
    out = torch.empty(4, 256, device="cuda", dtype=BF)
    for bad in (lambda: ops.linear_fp8(x[:, :100], wq, ws, status=st),
                lambda: ops.linear_fp8(x.double(), wq, ws, status=st),
                lambda: ops.linear_fp8(x[:, 1:], wq[:, 1:], ws, status=st),
                lambda: ops.linear_fp8(x, wq, ws[:1], status=st),
                lambda: ops.linear_fp8(x, wq, ws.double(), status=st),
                lambda: ops.linear_fp8(x, wq, ws, ws[0], status=st),
                lambda: ops.linear_fp8(x, wq, ws, torch.zeros(256, device="cuda", dtype=BF), status=st),
                lambda: ops.linear_fp8(x, wq, ws.cpu(), status=st),
                lambda: ops.linear_fp8(x, wq.cpu(), ws, status=st),
                lambda: ops.linear_fp8(x, x, ws, status=st),
                lambda: ops.linear_fp8(x, wq, ws, torch.zeros(256, device="cuda", requires_grad=True), status=st),
                lambda: ops.linear_fp8(x, wq, ws.clone().requires_grad_(), status=st),
                lambda: ops.gemm_fp8(xq, xs, wq, ws, out=out[:3]),
                lambda: ops.gemm_fp8(xq, xs, wq, ws, out=out.double()),
                lambda: ops.gemm_fp8(xq, xs, wq, ws, out=out.t()),
                lambda: ops.gemm_fp8(xq, xs.contiguous(), wq, ws),
                lambda: ops.gemm_fp8(xq, torch.ones(2, 5, device="cuda")[:, :4].T, wq, ws),
                lambda: ops.quantize_fp8(x, 2)):
        with pytest.raises((RuntimeError, ValueError)):
            bad()
    # twice differentiable it is not
    x = x.requires_grad_()
    y = ops.linear_fp8(x, wq, ws, status=st)
    g = torch.ones_like(y).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y, x, g, create_graph=True)
