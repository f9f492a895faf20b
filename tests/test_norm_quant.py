"""RMS norm with residual add and 8-bit output: statement on CPU, kernels against the definition in 64 bits, and the
operators of a frozen model in a row, up to the loss of the student that learns from it."""
import math

import pytest
import torch

from tests.test_int8 import U, check_quantised

# y of the kernels against 64 bits: the mean of squares is a chain of at most 60 positive additions and the rsqrt and
# three products follow: 60 / 2 + 4 + 3 roundings and less than 10 for the approximations
Y_SLACK = 50 * U


def exact(x, delta, w, eps, zero_centered=False):
    s = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    d = s.double()
    g = w.double() + (1.0 if zero_centered else 0.0)
    return s, d * torch.rsqrt(d.square().mean(-1, keepdim=True) + eps) * g


def check_e4m3(q, scale, y):
    b = y.view(y.shape[0], -1, 128)
    top = b.abs().amax(2)
    want = torch.where(top > 0, top / 448, 1.0)
    assert q.dtype == torch.float8_e4m3fn and ((scale.double() - want).abs() <= want * (Y_SLACK + 2 * U)).all()
    got = q.double().view(b.shape) * scale.double()[:, :, None]
    # half a step of e4m3 is 2^-4 of a normal value, 2^-10 of the scale below 2^-6 of it
    tol = b.abs() * (2.0 ** -4 + 4 * Y_SLACK) + want[:, :, None] * 2.0 ** -10 * (1 + 1e-5)
    assert ((got - b).abs() <= tol).all()


def make(T, H, device="cpu", dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g) * torch.rand(T, 1, generator=g).mul(6).exp()
    d = torch.randn(T, H, generator=g)
    w = 1 + 0.3 * torch.randn(H, generator=g)
    return [t.to(dtype).to(device) for t in (x, d, w)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_statement(dtype):
    from steptronoss_b200 import ops

    x, d, w = make(5, 256, dtype=dtype)
    for zc in (False, True):
        s, y = exact(x, d, w, 1e-5, zc)
        got, q, sc = ops.add_rmsnorm_quant(x.view(1, 5, 256), d.view(1, 5, 256), w, 1e-5, zc)
        assert got.shape == (1, 5, 256) and torch.equal(got[0], s) and q.shape == (5, 256)
        check_quantised(q, sc, y, 256 * U)
        _, q, sc = ops.add_rmsnorm_quant(x, d, w, 1e-5, zc, fmt="e4m3_1x128")
        check_e4m3(q, sc, y)
        q, sc = ops.rmsnorm_quant(x, w, 1e-5, zc)
        check_quantised(q, sc, exact(x, None, w, 1e-5, zc)[1], 256 * U)


def test_refusals():
    from steptronoss_b200 import ops

    x, d, w = make(3, 200)
    for args, kw, error in [((x, d, w), dict(fmt="fp4"), ValueError), ((x, d, w), dict(fmt="e4m3_1x128"), ValueError),
                            ((x, d[:2], w), {}, ValueError), ((x, d, w[:-1]), {}, ValueError),
                            ((x.float().requires_grad_(), d, w), {}, RuntimeError),
                            ((x, d, torch.nn.Parameter(w)), {}, RuntimeError)]:
        with pytest.raises(error):
            ops.add_rmsnorm_quant(*args, **kw)
    with torch.no_grad():
        ops.add_rmsnorm_quant(x, d, torch.nn.Parameter(w))
    s, q, sc = ops.add_rmsnorm_quant(x[:0], d[:0], w)
    assert s.shape == (0, 200) and q.shape == (0, 200) and sc.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(1, 1), (3, 7), (1, 4096), (5, 128), (130, 512), (67, 1000), (33, 1990), (9, 2048), (4, 5120),
                                 (3, 8192), (2, 8200), (2, 16384), (1, 32768), (2, 20001)])
def test_kernel_follows_the_definition(T, H):
    from steptronoss_b200 import ops

    x, d, w = make(T, H, "cuda")
    for zc in (False, True):
        s, y = exact(x, d, w, 1e-6, zc)
        got, q, sc = ops.add_rmsnorm_quant(x, d, w, 1e-6, zc)
        assert torch.equal(got, s) and q.stride(0) % 16 == 0
        check_quantised(q, sc, y, Y_SLACK)
        q, sc = ops.rmsnorm_quant(x, w, 1e-6, zc)
        check_quantised(q, sc, exact(x, None, w, 1e-6, zc)[1], Y_SLACK)
        if H % 128 == 0:
            got, q, sc = ops.add_rmsnorm_quant(x, d, w, 1e-6, zc, fmt="e4m3_1x128")
            assert torch.equal(got, s)
            check_e4m3(q, sc, y)


@pytest.mark.gpu
def test_residual_sum_of_any_two_magnitudes_is_rounded_once():
    from steptronoss_b200 import ops

    torch.manual_seed(3)
    T, H = 64, 4096
    x, d = ((torch.randn(T, H, device="cuda") * torch.randint(-30, 31, (T, H), device="cuda").float().exp2()).to(torch.bfloat16)
            for _ in range(2))
    d[:, ::3] = -x[:, ::3] * 1.0078125                        # near cancellation
    d[:, 1::7] = x[:, 1::7] * 2.0 ** -9                       # ties of the sum's last place
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    want = (x.double() + d.double()).to(torch.float32).to(torch.bfloat16)
    for fmt in ("int8", "e4m3_1x128"):
        s, _, _ = ops.add_rmsnorm_quant(x, d, w, fmt=fmt)
        assert torch.equal(s, want) and torch.equal(s, ops.add_rmsnorm(x, d, w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3_1x128"])
def test_strides_alignment_and_rows_without_numbers(fmt):
    from steptronoss_b200 import ops

    T, H = 6, 1280
    x, d, w = make(T, H, "cuda")
    x[1], d[1] = 0, 0                            # a row of zeros
    wide = torch.zeros(T, H + 11, dtype=torch.bfloat16, device="cuda")
    for first in (0, 8, 5):
        wide[:, first:first + H] = x
        back = d.t().contiguous().t()            # last dimension strided
        s, q, sc = ops.add_rmsnorm_quant(wide[:, first:first + H], back, w, fmt=fmt)
        want_s, y = exact(x, d, w, 1e-6)
        assert torch.equal(s, want_s) and sc[1].eq(1).all() and q[1].float().eq(0).all()
        (check_quantised if fmt == "int8" else check_e4m3)(q, sc, y, *([Y_SLACK] if fmt == "int8" else []))
    x[2, 1279] = math.nan
    x[3, 0] = math.inf
    s, q, sc = ops.add_rmsnorm_quant(x, d, w, fmt=fmt)
    assert sc[2].isnan().all() and sc[3].isnan().any() and sc[[0, 1, 4, 5]].isfinite().all()


@pytest.mark.gpu
def test_matches_the_bf16_operator_and_feeds_the_fp8_product():
    from steptronoss_b200 import ops
    from steptronoss_b200.ops import fp8, native

    x, d, w = make(300, 512, "cuda")
    s, y = ops.add_rmsnorm(x, d, w)
    s8, q, sc = ops.add_rmsnorm_quant(x, d, w, fmt="e4m3_1x128")
    assert torch.equal(s, s8)
    # both round the same fp32 values, to bf16 (2^-8) and to e4m3 (2^-4, or 2^-10 of the scale)
    tol = y.float().abs() * (2.0 ** -4 + 2.0 ** -7) + sc.repeat_interleave(128, 1) * 2.0 ** -10 * 1.01
    assert ((fp8.dequantize_rows(q, sc) - y.float()).abs() <= tol).all()
    wt = (torch.randn(256, 512, device="cuda") * 0.05).to(torch.bfloat16)
    wq, sw = fp8.quantize_blocks_128x128(wt)
    out = fp8.grouped_gemm_fp8(q, sc, wq, sw, None, 1)
    torch.cuda.synchronize()
    native.raise_if_kernel_error()
    want = fp8.dequantize_rows(q, sc).double() @ fp8.dequantize_blocks(wq, sw).double().t()
    size = fp8.dequantize_rows(q, sc).double().abs() @ fp8.dequantize_blocks(wq, sw).double().abs().t()
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 512 * U).all()


@pytest.mark.gpu
def test_a_student_learns_from_a_frozen_teacher_in_8_bits():
    """Residual add, norm to int8, the teacher's head in int8, its top logits, the student's fused head: in one go, and
    the same captured into a graph and replayed on new inputs."""
    from steptronoss_b200 import ops
    from steptronoss_b200.ops import native
    from tests.test_distillation import oracle

    torch.manual_seed(0)
    T, H, V, K = 200, 256, 4096, 16
    x, d, gain = make(T, H, "cuda")
    wq, sw = ops.quantize_rows_int8((torch.randn(V, H, device="cuda") * 0.2).to(torch.bfloat16))
    h = torch.randn(T, H, device="cuda").to(torch.bfloat16).requires_grad_()
    head = (torch.randn(V, H, device="cuda") * 0.1).to(torch.bfloat16).requires_grad_()
    weights = torch.full((T,), 1.0 / T, device="cuda")
    weights[::7] = 0

    def step():
        with torch.no_grad():
            _, q, sc = ops.add_rmsnorm_quant(x, d, gain)
            top, ids = ops.gemm_int8(q, sc, wq, sw, out_dtype=torch.float32).topk(K)
        total, tok = ops.fused_linear_topk_distillation(h, head, ids, top, weights, 2.0, chunk_tokens=64)
        return (total, tok, ids, top, *torch.autograd.grad(total, [h, head]))

    def verify(total, tok, ids, top, dh, dw):
        torch.cuda.synchronize()
        native.raise_if_kernel_error()
        _, q, sc = ops.add_rmsnorm_quant(x, d, gain)
        teacher = (q.double() * sc.double()[:, None]) @ (wq.double() * sw.double()[:, None]).t()
        assert ((teacher.gather(1, ids) - top.double()).abs() <= top.double().abs() * 4 * U + 1e-30).all()
        logits = h.detach().double() @ head.detach().double().t()
        want, grad, _, _ = oracle(logits, ids, top, 2.0, weights=weights)
        scale = float(logits.abs().max() + top.abs().max()) / 2
        assert (tok.double().cpu() - want).abs().max() <= (scale * 40 + 400) * U * 8
        for got, a, b in ((dh, grad, head.detach().double().cpu()), (dw, grad.t(), h.detach().double().cpu())):
            size = a.abs() @ b.abs()
            assert ((got.double().cpu() - a @ b).abs() <= size * 2.0 ** -7 + 1e-30).all()

    first = step()
    verify(*first)
    del first
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.mul_(0.5)
        h.mul_(-1.0)
    graph.replay()
    verify(*out)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3_1x128"])
def test_rows_up_to_the_largest_number(device, fmt):
    from steptronoss_b200 import ops

    g = torch.Generator().manual_seed(0)
    # values of one size, so that y = +-w (1 + at most 0.5) stays below 3.4e38
    x = ((torch.rand(3, 256, generator=g) + 1) * (torch.randint(0, 2, (3, 256), generator=g) * 2 - 1)).to(torch.bfloat16)
    w = ((torch.rand(256, generator=g) + 1) * 1e38).to(torch.bfloat16)
    x, d, w = x.to(device), torch.zeros_like(x).to(device), w.to(device)
    _, y = exact(x, d, w, 1e-6)
    assert 2.0 ** 126 < y.abs().amax() < 3.3e38
    _, q, sc = ops.add_rmsnorm_quant(x, d, w, fmt=fmt)
    (check_quantised if fmt == "int8" else check_e4m3)(q, sc, y, *([256 * U] if fmt == "int8" else []))


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(64, 512), (33, 4096), (5, 32768)])
def test_values_behind_the_norm_are_the_nearest_to_the_quotient(T, H):
    """With |s| = 1 throughout and eps = 0 the norm is exact: y = +-w."""
    from steptronoss_b200 import ops
    from steptronoss_b200.ops.int8 import quantize_rows_int8_reference

    torch.manual_seed(5)
    x = torch.randint(0, 2, (T, H), device="cuda").mul(2).sub(1).to(torch.bfloat16)
    w = (torch.randn(H, device="cuda") * torch.randint(-3, 4, (H,), device="cuda").float().exp2()).to(torch.bfloat16)
    w[0], w[1] = 32.0, 16.0
    y = (x.float() * w.float()).cpu()
    q, s = ops.rmsnorm_quant(x, w, 0.0)
    want, ws = quantize_rows_int8_reference(y)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), want)
    q, s = ops.rmsnorm_quant(x, w, 0.0, fmt="e4m3_1x128")
    b = y.view(T, H // 128, 128)
    top = b.abs().amax(2, keepdim=True)
    want = (448 * b.double() / top.double()).float().to(torch.float8_e4m3fn).view(T, H)
    assert torch.equal(s.cpu(), (top / 448).squeeze(2)) and torch.equal(q.float().cpu(), want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(64, 512), (4, 4096), (300, 4096), (100, 1280), (3, 32768)])
def test_e4m3_values_are_those_of_the_definition(T, H):
    """448 y / max|y| in real numbers: the norm's factor drops out, and 448 s w has 19 bits.  In 64 bits the quotient is off
    by 2^-51 of itself; one that lies on a border between two e4m3 values is put back there by the rounding to fp32, which
    any other is too far from (the numerator and the border times max|y| are integers of less than 30 bits)."""
    from steptronoss_b200 import ops

    x, d, w = make(T, H, "cuda")
    x[0, :128], d[0, :128] = x[0, :128].abs().log2().round().exp2(), 0              # powers of two
    s, y = exact(x, d, w, 1e-6)
    b = y.view(T, H // 128, 128)
    want = (448 * b / b.abs().amax(2, keepdim=True)).float().to(torch.float8_e4m3fn).view(T, H)
    _, q, sc = ops.add_rmsnorm_quant(x, d, w, 1e-6, fmt="e4m3_1x128")
    assert torch.equal(q.float(), want.float())
    check_e4m3(q, sc, y)
    q, _ = ops.rmsnorm_quant(s, w, 1e-6, fmt="e4m3_1x128")
    assert torch.equal(q.float(), want.float())
