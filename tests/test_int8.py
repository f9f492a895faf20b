"""8-bit integer products and row quantisation: the statements on CPU, the sm_100a kernels against the definition in
64 bits (the integer sums are exact, so only the roundings after them are allowed for)."""
import math

import pytest
import torch

U = 2.0 ** -24                      # one fp32 rounding


def operands(M, N, K, device, seed=0):
    """Values over the whole int8 range, -128 and 127 among them, in rows on 16-byte boundaries."""
    from steptronoss_b200.ops.int8 import pitched_like

    g = torch.Generator().manual_seed(seed)
    xq = torch.randint(-128, 128, (M, K), generator=g).to(torch.int8)
    wq = torch.randint(-128, 128, (N, K), generator=g).to(torch.int8)
    xq[0], wq[-1] = -128, -128      # the largest sum that there is
    sx, sw = torch.rand(M, generator=g) + 0.01, torch.rand(N, generator=g) * 0.02
    return [pitched_like(xq.to(device)), sx.to(device), pitched_like(wq.to(device)), sw.to(device)]


def check(y, xq, sx, wq, sw):
    exact = (xq.double() @ wq.double().t()) * sx.double()[:, None] * sw.double()[None]
    # int32 -> fp32, two multiplications, one rounding to the output's type
    tol = exact.abs() * (torch.finfo(y.dtype).eps / 2 + 4 * U) + 1e-30
    assert y.shape == exact.shape and ((y.double() - exact).abs() <= tol).all()


def check_quantised(q, scale, x, slack=2 * U):
    """`slack`: relative error of the values and of their maximum before the division."""
    x = x.double()
    top = x.abs().amax(1)
    want = torch.where(top > 0, top / 127, 1.0)
    assert q.dtype == torch.int8 and ((scale.double() - want).abs() <= want * (slack + 2 * U)).all()
    assert ((q.double() - x / want[:, None]).abs() <= 0.5 + 127 * (2 * slack + 4 * U)).all()


# --------------------------------------------------------------------------------------------------------- CPU
def test_statements():
    from steptronoss_b200 import ops

    torch.manual_seed(0)
    x = torch.randn(5, 37)
    x[2] = 0
    q, s = ops.quantize_rows_int8(x)
    check_quantised(q, s, x)
    assert s[2] == 1 and q[2].eq(0).all() and q.stride(0) % 16 == 0
    assert ((ops.dequantize_rows_int8(q, s) - x).abs() <= 0.5 * s[:, None] * (1 + 1e-6)).all()
    w = torch.randn(11, 37)
    wq, sw = ops.quantize_rows_int8(w)
    check(ops.gemm_int8(q, s, wq, sw), q, s, wq, sw)
    check(ops.gemm_int8(q, s, wq, sw, out_dtype=torch.float32), q, s, wq, sw)
    y = ops.linear_int8(x.view(5, 1, 37), wq, sw)
    assert y.shape == (5, 1, 11) and torch.equal(y.view(5, 11), ops.gemm_int8(q, s, wq, sw))
    out = torch.full((5, 13), 3.0)
    assert ops.gemm_int8(q, s, wq, sw, out=out[:, 1:12]).data_ptr() == out[:, 1:].data_ptr()
    assert out[:, 0].eq(3).all() and out[:, 12].eq(3).all()
    # |y| <= sum_k |x| |w|; each operand is off by half a step of its scale
    exact = x.double() @ w.double().t()
    tol = (0.51 * s.double()[:, None]) * w.double().abs().sum(1)[None] + 0.51 * sw.double()[None] * x.double().abs().sum(1)[:, None]
    tol = tol + 37 * 0.26 * s.double()[:, None] * sw.double()[None] + exact.abs() * 2.0 ** -8 + 1e-6
    assert ((y.view(5, 11).double() - exact).abs() <= tol * 1.01).all()


def test_rows_that_are_not_finite_stay_visible():
    from steptronoss_b200 import ops

    x = torch.ones(3, 8)
    x[1, 2], x[2, 3] = math.nan, math.inf
    q, s = ops.quantize_rows_int8(x)
    y = ops.gemm_int8(q, s, *ops.quantize_rows_int8(torch.ones(4, 8)))
    assert y[0].isfinite().all() and y[1:].isnan().all()


def test_refusals():
    from steptronoss_b200 import ops

    xq, sx, wq, sw = operands(3, 5, 16, "cpu")
    bad = [
        ((xq[:, :8], sx, wq, sw), {}, ValueError), ((xq.float(), sx, wq, sw), {}, TypeError),
        ((xq, sx[:2], wq, sw), {}, ValueError), ((xq, sx, wq, sw.double()), {}, ValueError),
        ((xq, sx[:, None], wq, sw), {}, ValueError), ((xq[0], sx, wq, sw), {}, ValueError),
        ((xq, sx, wq, sw), dict(out_dtype=torch.float16), TypeError),
        ((xq, sx, wq, sw), dict(out=torch.zeros(3, 4)), ValueError),
        ((xq, sx, wq, sw), dict(out=torch.zeros(5, 3).t()), ValueError),
        ((xq, sx, wq, sw), dict(out=torch.zeros(1, 5).expand(3, 5)), ValueError),
        ((xq[:, :0], sx, wq[:, :0], sw), {}, ValueError),
        ((torch.zeros(1, 131072, dtype=torch.int8), sx[:1], torch.zeros(1, 131072, dtype=torch.int8), sw[:1]), {}, ValueError),
    ]
    for args, kw, error in bad:
        with pytest.raises(error):
            ops.gemm_int8(*args, **kw)
    x = torch.zeros(3, 16, requires_grad=True)
    for call in (lambda: ops.linear_int8(x, wq, sw), lambda: ops.quantize_rows_int8(x)):
        with pytest.raises(RuntimeError):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(ValueError):
        ops.quantize_rows_int8(torch.zeros(3))
    with pytest.raises(ValueError):
        ops.quantize_rows_int8(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        ops.linear_int8(torch.zeros(3, 8), wq, sw)


def test_no_tokens_and_no_channels():
    from steptronoss_b200 import ops

    xq, sx, wq, sw = operands(3, 5, 16, "cpu")
    assert ops.gemm_int8(xq[:0], sx[:0], wq, sw).shape == (0, 5)
    assert ops.linear_int8(torch.zeros(0, 16), wq, sw).shape == (0, 5)
    assert ops.gemm_int8(xq, sx, wq[:0], sw[:0]).shape == (3, 0)


# --------------------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 128, 128), (2, 7, 15), (16, 129, 100), (1, 6144, 4096), (17, 1000, 129), (33, 640, 2050), (64, 2051, 5000),
    (65, 256, 1024), (100, 4100, 300), (128, 128, 12288), (129, 4104, 256), (515, 2051, 1990), (300, 20000, 16),
    (1000, 9000, 300), (2000, 9001, 260), (2050, 9008, 129), (4000, 10000, 384), (1, 300, 131071),
])
def test_product_is_exact_up_to_the_last_roundings(M, N, K):
    from steptronoss_b200 import ops
    from steptronoss_b200.ops import native

    xq, sx, wq, sw = operands(M, N, K, "cuda")
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((M, N + 24), 7.0, dtype=dtype, device="cuda")
        for first in (0, 8, 3):                       # aligned rows, shifted aligned rows, rows on odd addresses
            wide.fill_(7.0)
            y = ops.gemm_int8(xq, sx, wq, sw, out=wide[:, first:first + N])
            torch.cuda.synchronize()
            native.raise_if_kernel_error()
            check(y, xq, sx, wq, sw)
            assert wide[:, :first].eq(7).all() and wide[:, first + N:].eq(7).all()
        y2 = ops.gemm_int8(xq, sx, wq, sw, out_dtype=dtype)
        assert torch.equal(y, y2)


@pytest.mark.gpu
def test_rows_behind_the_last_token_stay():
    from steptronoss_b200 import ops

    for M in (1, 40, 700):
        xq, sx, wq, sw = operands(M + 20, 9000, 256, "cuda")
        y = torch.full((M + 20, 9000), 5.0, dtype=torch.bfloat16, device="cuda")
        ops.gemm_int8(xq[:M], sx[:M], wq, sw, out=y[:M])
        check(y[:M], xq[:M], sx[:M], wq, sw)
        assert y[M:].eq(5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(20000, 110000), (129, 17000000)])
def test_more_results_than_32_bits_count(M, N):
    from steptronoss_b200 import ops

    assert M * N > 2 ** 31
    xq, sx, wq, sw = operands(M, 64, 32, "cuda")
    wq, sw = wq.repeat((N + 63) // 64, 1)[:N], sw.repeat((N + 63) // 64)[:N].contiguous()
    y = ops.gemm_int8(xq, sx, wq, sw)
    for rows in (slice(0, 2), slice(M - 2, M)):
        for cols in (slice(0, 200), slice(N - 200, N)):
            check(y[rows, cols], xq[rows], sx[rows], wq[cols], sw[cols])


@pytest.mark.gpu
def test_a_single_row_needs_no_pitch():
    from steptronoss_b200 import ops

    xq, sx, wq, sw = operands(1, 300, 100, "cuda")
    flat = torch.empty(1, 100, dtype=torch.int8, device="cuda").copy_(xq)
    assert flat.stride(0) == 100
    check(ops.gemm_int8(flat, sx, wq, sw), xq, sx, wq, sw)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(1, 1), (1, 8), (3, 7), (300, 128), (5, 1990), (77, 2050), (9, 4096), (4, 12288), (2, 32768),
                                 (3, 20001)])
def test_quantised_rows(M, K):
    from steptronoss_b200 import ops

    torch.manual_seed(0)
    x = (torch.randn(M, K + 5, device="cuda") * torch.rand(M, 1, device="cuda").mul(8).exp()).to(torch.bfloat16)
    for view in (x[:, :K].contiguous(), x[:, 3:3 + K]):
        q, s = ops.quantize_rows_int8(view)
        check_quantised(q, s, view)
    z = x[:, :K].clone()
    z[0] = 0
    q, s = ops.quantize_rows_int8(z)
    assert s[0] == 1 and q[0].eq(0).all()
    z[0, K // 2] = math.nan
    if M > 1:
        z[1, K - 1] = -math.inf
    q, s = ops.quantize_rows_int8(z)
    assert s[:2].isnan().all() and s[2:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 1000, 512), (40, 640, 1990), (1333, 5001, 2050)])
def test_linear_on_the_fly(M, N, K):
    from steptronoss_b200 import ops

    torch.manual_seed(1)
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    wq, sw = ops.quantize_rows_int8((torch.randn(N, K, device="cuda") * 0.02).to(torch.bfloat16))
    y = ops.linear_int8(x.view(1, M, K), wq, sw)
    q, s = ops.quantize_rows_int8(x)
    check(y.view(M, N), q, s, wq, sw)


@pytest.mark.gpu
def test_products_on_two_streams_and_in_a_graph():
    from steptronoss_b200 import ops

    sets = [operands(m, 6144, 2048, "cuda", seed=m) for m in (3, 500)]
    want = [ops.gemm_int8(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    torch.cuda.synchronize()
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append([ops.gemm_int8(*s) for _ in range(4)])
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(a, y) for a in ys)
    x = torch.randn(3, 2048, device="cuda").to(torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_int8(x, sets[0][2], sets[0][3])
    x.mul_(-2)
    want = ops.linear_int8(x, sets[0][2], sets[0][3])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 700])
def test_kernels_that_follow_each_other_wait_for_their_operands(M):
    """Each kernel may be set up while the one before it runs; tokens, weights and results are made and used in a row, the
    same memory again and again."""
    from steptronoss_b200 import ops

    torch.manual_seed(5)
    N, K, rounds = 3000, 1536, 12
    xs = [torch.randn(M, K, device="cuda").to(torch.bfloat16) for _ in range(rounds)]
    ws = [torch.randn(N, K, device="cuda").to(torch.bfloat16) for _ in range(rounds)]
    gain = torch.ones(K, dtype=torch.bfloat16, device="cuda")

    def one(x, w):
        wq, sw = ops.quantize_rows_int8(w)
        s, q, sq = ops.add_rmsnorm_quant(x, x, gain)
        y = ops.gemm_int8(q, sq, wq, sw)
        y2 = ops.linear_int8(y[:, :K], wq, sw)
        return s, y, y2

    want = []
    for x, w in zip(xs, ws):
        torch.cuda.synchronize()
        wq, sw = ops.quantize_rows_int8(w)
        torch.cuda.synchronize()
        s, q, sq = ops.add_rmsnorm_quant(x, x, gain)
        torch.cuda.synchronize()
        y = ops.gemm_int8(q, sq, wq, sw)
        torch.cuda.synchronize()
        q2, s2 = ops.quantize_rows_int8(y[:, :K])
        torch.cuda.synchronize()
        want.append((s, y, ops.gemm_int8(q2, s2, wq, sw)))
    torch.cuda.synchronize()
    for _ in range(3):
        got = [one(x, w) for x, w in zip(xs, ws)]
        assert all(torch.equal(a, b) for g, t in zip(got, want) for a, b in zip(g, t))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [one(x, w) for x, w in zip(xs, ws)]
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for g, t in zip(got, want) for a, b in zip(g, t))


@pytest.mark.gpu
def test_kernels_behind_a_fork_and_a_join_of_streams():
    """A product directly behind an event that another stream recorded, eagerly and in a captured graph."""
    from steptronoss_b200 import ops

    xq, sx, wq, sw = operands(33, 4096, 2048, "cuda", seed=7)
    x = torch.randn(33, 2048, device="cuda").to(torch.bfloat16)
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")

    def work():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            slow = big @ big                                     # keeps the side stream busy before it quantises
            q, s = ops.quantize_rows_int8(x + (slow[:33, :2048] * 0).to(torch.bfloat16))
        first = ops.gemm_int8(xq, sx, wq, sw)
        main.wait_stream(side)
        second = ops.gemm_int8(q, s, wq, sw)                     # right behind the join
        for t in (slow, q, s):
            t.record_stream(main)
        return first, second

    want = ops.gemm_int8(xq, sx, wq, sw), ops.linear_int8(x, wq, sw)
    torch.cuda.synchronize()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(work(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_gpu_refusals():
    from steptronoss_b200 import ops

    xq, sx, wq, sw = operands(3, 5, 100, "cuda")
    with pytest.raises(ValueError):
        ops.gemm_int8(xq.contiguous(), sx, wq, sw)                 # a pitch of 100 bytes
    with pytest.raises(ValueError):
        ops.gemm_int8(xq[:, 1:], sx, wq[:, 1:], sw)                # rows that start one byte off
    with pytest.raises(ValueError):
        ops.gemm_int8(xq, sx.cpu(), wq, sw)
    with pytest.raises(TypeError):
        ops.quantize_rows_int8(torch.zeros(3, 16, device="cuda"))
    with pytest.raises(ValueError):
        ops.quantize_rows_int8(torch.zeros(1, 32769, dtype=torch.bfloat16, device="cuda"))


LARGE = [8.5e37, 8.6e37, 1.2e38, 3.3895e38]      # around 2^126 and up to the largest bf16


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("K", [8, 129, 1990])
def test_rows_up_to_the_largest_number(device, K):
    from steptronoss_b200 import ops

    g = torch.Generator().manual_seed(0)
    x = torch.rand(len(LARGE), K, generator=g) * 2 - 1
    x[:, K // 2] = 1.0
    x = (x * torch.tensor(LARGE)[:, None]).to(torch.bfloat16).to(device)
    assert x.isfinite().all()
    q, s = ops.quantize_rows_int8(x)
    assert q[:, K // 2].eq(127).all()
    check_quantised(q, s, x)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(2000, 512), (700, 1990), (300, 4096), (9, 20001)])
def test_values_are_the_nearest_to_the_quotient_by_the_stored_scale(M, K):
    """bf16 rows are full of quotients that lie on a border between two values (rows whose largest value is a power of two
    have 63.5 steps at its half), so the division has to be the one that the definition makes."""
    from steptronoss_b200 import ops
    from steptronoss_b200.ops.int8 import quantize_rows_int8_reference

    torch.manual_seed(4)
    x = (torch.randn(M, K, device="cuda") * torch.rand(M, 1, device="cuda").mul(60).sub(30).exp2()).to(torch.bfloat16)
    x[::3, 5] = x[::3].float().abs().amax(1).log2().ceil().exp2().to(torch.bfloat16)     # largest value a power of two
    x[::3, 6] = x[::3, 5] / 2
    q, s = ops.quantize_rows_int8(x)
    want, ws = quantize_rows_int8_reference(x.cpu())               # where / is a division
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 5, 40, 100, 700])
def test_scales_written_by_the_kernel_before(M):
    """The same memory holds other scales in every round; the product that reads them is set up while they are written."""
    from steptronoss_b200 import ops

    torch.manual_seed(6)
    N, K, rounds = 1500, 768, 30
    wq, sw = ops.quantize_rows_int8(torch.randn(N, K, device="cuda").to(torch.bfloat16))
    xs = [(torch.randn(M, K, device="cuda") * 2.0 ** (r % 13 - 6)).to(torch.bfloat16) for r in range(rounds)]
    want = []
    for x in xs:
        q, s = ops.quantize_rows_int8(x)
        torch.cuda.synchronize()
        want.append(ops.gemm_int8(q, s, wq, sw))
        torch.cuda.synchronize()
    for _ in range(3):
        got = [ops.linear_int8(x, wq, sw) for x in xs]         # freed scales come back in the next round
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.empty_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_int8(x, wq, sw)
    for src, ref in zip(xs, want):
        x.copy_(src)
        graph.replay()
        assert torch.equal(y, ref)


@pytest.mark.parametrize("M, N", [(2 ** 30 + 1, 1), (1, 2 ** 31 + 1), (2 ** 32 + 3, 1)])
def test_sizes_beyond_the_kernels_are_refused(M, N):
    """Sizes cross the C interface as 32-bit numbers: larger ones would be taken for smaller ones there."""
    from steptronoss_b200 import ops

    row = lambda n: torch.zeros(1, 16, dtype=torch.int8).expand(n, 16)
    scale = lambda n: torch.ones(1).expand(n)
    with pytest.raises(ValueError, match="at most"):
        ops.gemm_int8(row(M), scale(M), row(N), scale(N))
    with pytest.raises(ValueError, match="at most"):
        ops.linear_int8(torch.zeros(1, 16).expand(M, 16) if M > 1 else torch.zeros(1, 16), row(N), scale(N))
