"""Distillation from a teacher's top logits: the statement on CPU, two vocabulary shards on gloo ranks, and the sm_100a
kernels against the definition in 64 bits."""
import math
import os

import pytest
import torch
import torch.multiprocessing as mp

from tests.dist_helpers import free_port

INF = math.inf


def oracle(logits, ids, teacher, tau, vocab=None, weights=None):
    """Loss [T], gradient [T, V] of sum_t w_t loss_t, p and q per token, from the definition, in 64 bits."""
    s = logits.double().cpu() / tau
    T, V = s.shape
    t = teacher.double().cpu() / tau
    ids = ids.long().cpu()
    w = torch.ones(T, dtype=torch.float64) if weights is None else weights.double().cpu()
    inside = (ids >= 0) & (ids < (vocab or V))
    t = torch.where(inside, t, -INF)
    loss = torch.zeros(T, dtype=torch.float64)
    q_all = torch.zeros(T, V, dtype=torch.float64)
    logp = torch.log_softmax(s, -1)
    p = logp.exp()
    has = torch.zeros(T, dtype=torch.bool)
    for r in range(T):
        keep = t[r] > -INF
        if not keep.any():
            continue
        has[r] = True
        logq = torch.log_softmax(t[r][keep], -1)
        q = logq.exp()
        i = ids[r][keep]
        d = logq - logp[r][i]
        loss[r] = (q * torch.where(q > 0, d, 0.0)).sum()
        q_all[r].index_add_(0, i, q)
    live = (has & (w != 0)).unsqueeze(1)
    grad = torch.where(live, (p - q_all) / tau * w.unsqueeze(1), 0.0)
    return loss, grad, p, q_all


def bounds(logits, teacher, tau, p, q, grad, w, out_dtype):
    """Largest error of loss and gradient by arithmetic, u = 2^-24 per fp32 rounding.  Exponents in units of log2 reach
    A; an exponent of size A is off by 2 A u after its products, ex2 and lg2 by 4 u; a row's sum is a chain of at most
    200 additions.  So p is off by (2A + 212) u of itself, q by (2A + 48) u, the logarithms by (4A + 212) u, and q
    enters the loss times a difference of logarithms of at most 2A."""
    u = 2.0 ** -24
    fin = lambda x: x.double()[torch.isfinite(x.double())]
    span = lambda x: float((x.max() - x.min())) if x.numel() else 0.0
    A = 1.4427 * max(span(fin(logits)), span(fin(teacher)), float(fin(logits).abs().max()), 1.0) / tau + 20
    ep, eq = (2 * A + 212) * u, (2 * A + 48) * u
    loss_tol = (4 * A + 212) * u + 2 * A * eq
    half_step = torch.finfo(out_dtype).eps / 2
    grad_tol = w.abs().unsqueeze(1) / tau * (p * ep + q * eq) * 1.01 + grad.abs() * half_step + 1e-37
    return loss_tol, grad_tol


def make(T, V, K, seed=0, dtype=torch.float32, device="cpu", spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, V, generator=g) * spread).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]) if K <= V else torch.randint(
        0, V, (T, K), generator=g)
    teacher = torch.randn(T, K, generator=g) * spread
    weights = torch.rand(T, generator=g) + 0.5
    return [x.to(device) for x in (logits, ids, teacher, weights)]


def check(loss, grad, logits, ids, teacher, weights, tau):
    want, wgrad, p, q = oracle(logits, ids, teacher, tau, weights=weights)
    loss_tol, grad_tol = bounds(logits.cpu(), teacher.cpu(), tau, p, q, wgrad, weights.double().cpu(), grad.dtype)
    assert loss.dtype == torch.float32
    assert (loss.double().cpu() - want).abs().max() <= loss_tol
    assert ((grad.double().cpu() - wgrad).abs() <= grad_tol).all()


# --------------------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("tau", [1.0, 0.5, 4.0])
def test_statement_follows_the_definition(tau):
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(7, 53, 6)
    teacher[1, 3:] = -INF                 # a shorter row
    teacher[2] = -INF                     # a row without entries
    ids[3, 1] = ids[3, 0]                 # the same id twice
    ids[4, 2], ids[4, 3] = -1, 53         # ids outside the vocabulary
    w[5] = 0.0
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w, tau)
    check(loss, grad, logits, ids, teacher, w, tau)
    assert loss[2] == 0 and grad[2].eq(0).all() and grad[5].eq(0).all()
    x = logits.clone().requires_grad_()
    per_token = topk_distillation(x, ids, teacher, tau)
    (per_token * w).sum().backward()
    assert torch.equal(per_token.detach(), loss) and torch.allclose(x.grad, grad, atol=1e-7)
    lead = topk_distillation(logits.view(1, 7, 53), ids.view(1, 7, 6), teacher.view(1, 7, 6), tau)
    assert lead.shape == (1, 7) and torch.equal(lead[0], loss)


def test_gradient_agrees_with_differences():
    from steptronoss_b200.ops import topk_distillation

    logits, ids, teacher, _ = make(4, 11, 5, dtype=torch.float64)
    ids[0, 1] = ids[0, 0]
    teacher[1, 2:] = -INF
    torch.autograd.gradcheck(lambda x: topk_distillation(x, ids, teacher, 1.5), logits.requires_grad_(), atol=1e-6)


def test_rows_that_do_not_count_may_hold_anything():
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(4, 9, 3)
    logits[0], logits[1, 2] = math.nan, -INF
    teacher[0] = -INF
    logits[2] = math.nan
    w[2] = 0.0
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    assert loss[0] == 0 and grad[0].eq(0).all() and grad[2].eq(0).all() and grad[1].isfinite().all()
    x = logits.clone().requires_grad_()
    loss = topk_distillation(x, ids, teacher)
    loss[torch.tensor([0, 1, 3])].sum().backward()
    assert x.grad[0].eq(0).all() and x.grad[2].eq(0).all() and x.grad.isfinite().all()


def test_a_teacher_that_is_not_a_number_shows_in_its_token_alone():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(3, 9, 3)
    teacher[1, 0], teacher[1, 2], ids[1] = math.nan, -INF, torch.tensor([4, 5, 0])
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    assert loss[1].isnan() and loss[[0, 2]].isfinite().all() and grad[[0, 2]].isfinite().all()
    assert grad[1, 4].isnan() and grad[1, 5].isnan() and grad[1, 0].isfinite()


def test_zero_entries_and_zero_tokens():
    from steptronoss_b200.ops import fused_linear_topk_distillation, topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(3, 9, 2)
    loss, grad = topk_distillation_loss_and_grad(logits, ids[:, :0], teacher[:, :0], w)
    assert loss.eq(0).all() and grad.eq(0).all()
    loss, grad = topk_distillation_loss_and_grad(logits[:0], ids[:0], teacher[:0], w[:0])
    assert loss.shape == (0,) and grad.shape == (0, 9)
    total, tok = fused_linear_topk_distillation(torch.zeros(0, 8), torch.zeros(16, 8), ids[:0], teacher[:0], w[:0])
    assert total == 0 and tok.shape == (0,)


def test_in_place_and_given_output():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(5, 33, 4)
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    wide = torch.full((5, 40), 7.0, dtype=torch.bfloat16)
    loss2, out = topk_distillation_loss_and_grad(logits, ids, teacher, w, out=wide[:, :33])
    assert torch.equal(loss, loss2) and torch.equal(out, grad.to(torch.bfloat16)) and wide[:, 33:].eq(7).all()
    buf = logits.clone()
    loss3, out = topk_distillation_loss_and_grad(buf, ids, teacher, w, out=buf)
    assert out.data_ptr() == buf.data_ptr() and torch.equal(loss, loss3) and torch.equal(buf, grad)


def test_fused_head_on_cpu_is_the_head_and_the_loss():
    from steptronoss_b200.ops import fused_linear_topk_distillation, topk_distillation

    torch.manual_seed(0)
    _, ids, teacher, w = make(6, 24, 4)
    h, head = torch.randn(6, 8, requires_grad=True), torch.randn(24, 8, requires_grad=True)
    total, tok = fused_linear_topk_distillation(h, head, ids, teacher, w, 2.0)
    got = torch.autograd.grad(total, [h, head])
    loss = topk_distillation(h @ head.t(), ids, teacher, 2.0)
    want = torch.autograd.grad((loss * w).sum(), [h, head])
    assert torch.allclose(tok, loss) and not tok.requires_grad
    assert all(torch.allclose(a, b, atol=1e-6) for a, b in zip(got, want))


@pytest.mark.parametrize("change, error", [
    (dict(teacher_ids=torch.zeros(4, 3, dtype=torch.long)), ValueError),
    (dict(teacher_logits=torch.zeros(3, 2)), ValueError),
    (dict(teacher_ids=torch.zeros(4, 2)), TypeError),
    (dict(teacher_logits=torch.zeros(4, 2, dtype=torch.long)), TypeError),
    (dict(teacher_logits=torch.zeros(4, 2, requires_grad=True)), ValueError),
    (dict(teacher_ids=torch.zeros(4, 1025, dtype=torch.long), teacher_logits=torch.zeros(4, 1025)), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=-1.0), ValueError),
    (dict(temperature=math.nan), ValueError),
    (dict(temperature=math.inf), ValueError),
    (dict(temperature=1e-7), ValueError),
    (dict(temperature=1e7), ValueError),
    (dict(weights=torch.ones(3)), ValueError),
    (dict(logits=torch.zeros(2, 2, 9)), ValueError),
    (dict(logits=torch.zeros(4, 0)), ValueError),
    (dict(out=torch.zeros(4, 8)), ValueError),
    (dict(out=torch.zeros(4, 9, dtype=torch.float16)), TypeError),
    (dict(out=torch.zeros(9, 4).t()), ValueError),
    (dict(out=torch.zeros(1, 9).expand(4, 9)), ValueError),
    (dict(out=torch.zeros(4, 9, requires_grad=True)), ValueError),
])
def test_refusals(change, error):
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    args = dict(logits=torch.zeros(4, 9), teacher_ids=torch.zeros(4, 2, dtype=torch.long),
                teacher_logits=torch.zeros(4, 2), weights=torch.ones(4))
    topk_distillation_loss_and_grad(**args)
    with pytest.raises(error):
        topk_distillation_loss_and_grad(**{**args, **change})


def test_refuses_an_output_that_overlaps_the_logits():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    buf = torch.zeros(100)
    logits, out = buf[:36].view(4, 9), buf[4:40].view(4, 9)
    with pytest.raises(ValueError):
        topk_distillation_loss_and_grad(logits, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2), torch.ones(4), out=out)


def test_refuses_a_shard_outside_the_vocabulary():
    from steptronoss_b200.ops import fused_linear_topk_distillation, topk_distillation

    ids, t = torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)
    for start in (-1, 1, 9):
        with pytest.raises(ValueError):
            topk_distillation(torch.zeros(4, 9), ids, t, 1.0, start)
        with pytest.raises(ValueError):
            fused_linear_topk_distillation(torch.zeros(4, 8), torch.zeros(16, 8), ids, t, torch.ones(4), 1.0, start)


def test_second_derivatives_are_refused():
    from steptronoss_b200.ops import topk_distillation

    logits, ids, teacher, _ = make(3, 9, 2)
    loss = topk_distillation(logits.requires_grad_(), ids, teacher).sum()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, logits, create_graph=True)


def test_fused_head_refuses_weights_that_want_a_gradient():
    from steptronoss_b200.ops import fused_linear_topk_distillation

    _, ids, teacher, w = make(3, 64, 2)
    h, head = torch.zeros(3, 16), torch.zeros(64, 16)
    with pytest.raises(ValueError, match="no gradient flows to the weights"):
        fused_linear_topk_distillation(h, head, ids, teacher, w.requires_grad_())
    with torch.no_grad():
        fused_linear_topk_distillation(h, head, ids, teacher, w)


def test_fused_head_refusals():
    from steptronoss_b200.ops import fused_linear_topk_distillation as f

    ids, t, w = torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2), torch.ones(4)
    for h, head, more in ((torch.zeros(4, 8), torch.zeros(16, 7), {}), (torch.zeros(1, 4, 8), torch.zeros(16, 8), {}),
                          (torch.zeros(4, 8), torch.zeros(16, 8), dict(chunk_tokens=0)),
                          (torch.zeros(5, 8), torch.zeros(16, 8), {})):
        with pytest.raises(ValueError):
            f(h, head, ids, t, w, **more)


def _shard_worker(rank, world, port, q):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1",
                      MASTER_PORT=str(port))
    torch.set_num_threads(1)
    try:
        import torch.distributed as dist

        from steptronoss_b200.ops import topk_distillation

        dist.init_process_group("gloo", rank=rank, world_size=world)
        logits, ids, teacher, w = make(6, 16, 5, seed=3)
        teacher[1, 2:] = -INF
        teacher[2] = -INF
        ids[3, 0], ids[4, 1] = 99, ids[4, 0]
        shard = logits[:, rank * 8:(rank + 1) * 8].clone().requires_grad_()
        loss = topk_distillation(shard, ids, teacher, 2.0, rank * 8, dist.group.WORLD)
        (loss * w).sum().backward()
        q.put((rank, loss.tolist(), shard.grad.tolist(), None))
        dist.barrier()
        dist.destroy_process_group()
    except BaseException:
        import traceback

        q.put((rank, None, None, traceback.format_exc()))
        raise


def test_two_vocabulary_shards_equal_the_whole():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = free_port()
    procs = [ctx.Process(target=_shard_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = {}
    try:
        for _ in range(2):
            rank, loss, grad, err = q.get(timeout=120)
            assert err is None, err
            res[rank] = (torch.tensor(loss), torch.tensor(grad))
    finally:
        for p in procs:
            p.join(timeout=30)
            if p.is_alive():
                p.kill()
    logits, ids, teacher, w = make(6, 16, 5, seed=3)
    teacher[1, 2:] = -INF
    teacher[2] = -INF
    ids[3, 0], ids[4, 1] = 99, ids[4, 0]
    check(res[0][0], torch.cat([res[0][1], res[1][1]], dim=1), logits, ids, teacher, w, 2.0)
    assert torch.equal(res[0][0], res[1][0])


# --------------------------------------------------------------------------------------------------------- GPU
SHAPES = [(1, 1, 1), (3, 7, 3), (5, 1000, 17), (70, 4099, 33), (2, 50257, 20), (149, 2048, 64), (3, 151936, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,K", SHAPES)
def test_one_pass_kernel_follows_the_definition(T, V, K, dtype):
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    for tau, id_type in ((1.0, torch.int64), (0.5, torch.int32)):
        logits, ids, teacher, w = make(T, V, K, dtype=dtype, device="cuda")
        loss, grad = topk_distillation_loss_and_grad(logits, ids.to(id_type), teacher, w, tau)
        assert grad.dtype == dtype
        check(loss, grad, logits, ids, teacher, w, tau)
        again, grad2 = topk_distillation_loss_and_grad(logits, ids.to(id_type), teacher, w, tau)
        assert torch.equal(loss, again) and torch.equal(grad, grad2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,K", SHAPES)
def test_autograd_kernels_follow_the_definition(T, V, K, dtype):
    from steptronoss_b200.ops import topk_distillation

    logits, ids, teacher, w = make(T, V, K, seed=1, dtype=dtype, device="cuda")
    x = logits.clone().requires_grad_()
    loss = topk_distillation(x.view(1, T, V), ids.view(1, T, K), teacher.view(1, T, K), 2.0)
    (grad,) = torch.autograd.grad(loss, x, w.view(1, T))
    check(loss.detach().view(T), grad, logits, ids, teacher, w, 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,V", [(torch.bfloat16, 1501, 2001), (torch.float32, 999, 501), (torch.bfloat16, 401, 60000),
                                       (torch.float32, 333, 50257), (torch.float32, 150, 151936)])
def test_more_rows_than_run_at_a_time(dtype, T, V):
    """Running clusters take over the rows of clusters that have not started: with 1, 2, 4 and 8 CTAs each."""
    from steptronoss_b200.ops import native, topk_distillation, topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(T, V, 9, seed=9, dtype=dtype, device="cuda")
    teacher[::7, 4:] = -INF
    teacher[::11] = -INF
    ids[::5, 1] = ids[::5, 0]
    want, wgrad, p, q = oracle(logits, ids, teacher, 1.0, weights=w)
    loss_tol, grad_tol = bounds(logits.cpu(), teacher.cpu(), 1.0, p, q, wgrad, w.double().cpu(), dtype)
    for _ in range(3):
        loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
        torch.cuda.synchronize()
        native.raise_if_kernel_error()
        assert (loss.double().cpu() - want).abs().max() <= loss_tol
        assert ((grad.double().cpu() - wgrad).abs() <= grad_tol).all()
    # the loss alone and the backward pass take a whole row in one CTA where there are many rows
    x = logits.clone().requires_grad_()
    for _ in range(2):
        tok = topk_distillation(x, ids, teacher)
        (grad2,) = torch.autograd.grad(tok, x, w)
        torch.cuda.synchronize()
        native.raise_if_kernel_error()
        assert (tok.detach().double().cpu() - want).abs().max() <= loss_tol
        assert ((grad2.double().cpu() - wgrad).abs() <= grad_tol).all()
    buf = logits.clone()
    assert torch.equal(topk_distillation_loss_and_grad(buf, ids, teacher, w, out=buf)[0], loss) and torch.equal(buf, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_repeated_and_foreign_ids_on_the_gpu(dtype):
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    T, V, K = 9, 20000, 40
    logits, ids, teacher, w = make(T, V, K, seed=2, dtype=dtype, device="cuda")
    teacher[1, 5:] = -INF
    teacher[2] = -INF
    ids[3, 7:20] = ids[3, 6]                       # thirteen entries of one id
    ids[4, 0], ids[4, 1], ids[4, 2] = -1, V, 2 ** 40
    w[5] = 0.0
    logits[6, 100:300] = -INF                      # a masked part of the vocabulary, no entry there
    ids[6] = torch.arange(1000, 1000 + K, device="cuda")
    ids[7, 0], ids[7, 1] = 0, V - 1                # the ends of a row
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    check(loss, grad, logits, ids, teacher, w, 1.0)
    assert loss[2] == 0 and grad[2].eq(0).all() and grad[5].eq(0).all() and grad[6, 100:300].eq(0).all()
    x = logits.clone().requires_grad_()
    tok = topk_distillation(x, ids, teacher)
    (grad2,) = torch.autograd.grad(tok, x, w)
    check(tok.detach(), grad2, logits, ids, teacher, w, 1.0)
    # rows that do not count may hold anything; a NaN elsewhere stays in its row and shows
    logits[2] = math.nan
    logits[5, 3] = math.nan
    logits[8, 4] = math.nan
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    assert loss[2] == 0 and grad[2].eq(0).all() and grad[5].eq(0).all()
    assert loss[8].isnan() and grad[8].isnan().all()
    rest = [0, 1, 3, 4, 6, 7]
    assert loss[rest].isfinite().all() and grad[rest].isfinite().all()


@pytest.mark.gpu
def test_a_teacher_that_is_not_a_number_on_the_gpu():
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(3, 900, 3, device="cuda")
    teacher[1, 0], teacher[1, 2], ids[1] = math.nan, -INF, torch.tensor([4, 5, 0], device="cuda")
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    x = logits.clone().requires_grad_()
    tok = topk_distillation(x, ids, teacher)
    for l, g in ((loss, grad), (tok.detach(), torch.autograd.grad(tok, x, w)[0])):
        assert l[1].isnan() and l[[0, 2]].isfinite().all() and g[[0, 2]].isfinite().all()
        assert g[1, 4].isnan() and g[1, 5].isnan() and g[1, 0].isfinite() and g[1, 6:].isfinite().all()


@pytest.mark.gpu
def test_infinite_loss_where_the_student_excludes_an_entry():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(2, 600, 4, device="cuda")
    logits[0, ids[0, 1]] = -INF
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    assert loss[0] == INF and loss[1].isfinite() and grad.isfinite().all()
    q = torch.softmax(teacher[0].double(), 0)[1]
    assert abs(float(grad[0, ids[0, 1]]) + float(q * w[0])) < 1e-6       # p = 0 there
    logits[1] = -INF
    assert topk_distillation_loss_and_grad(logits, ids, teacher, w)[0][1].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_alignment_and_in_place(dtype):
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    T, V, K = 6, 5003, 12
    logits, ids, teacher, w = make(T, V, K, seed=4, dtype=dtype, device="cuda")
    want_loss, want = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    for pitch, first in ((5008, 0), (5011, 3), (5024, 1)):
        store = torch.full((T * pitch + 8,), 5.0, dtype=dtype, device="cuda")
        view = store[first:first + T * pitch].view(T, pitch)[:, :V]
        view.copy_(logits)
        out_store = torch.full((T, V + 9), 3.0, dtype=dtype, device="cuda")
        loss, grad = topk_distillation_loss_and_grad(view, ids, teacher, w, out=out_store[:, 2:2 + V])
        check(loss, grad, logits, ids, teacher, w, 1.0)
        assert out_store[:, :2].eq(3).all() and out_store[:, 2 + V:].eq(3).all()
        if dtype == torch.float32:
            half = torch.full((T, V + 5), 3.0, dtype=torch.bfloat16, device="cuda")
            loss, grad = topk_distillation_loss_and_grad(view, ids, teacher, w, out=half[:, 1:1 + V])
            check(loss, grad, logits, ids, teacher, w, 1.0)
            assert half[:, 0].eq(3).all() and half[:, 1 + V:].eq(3).all()
        x = view.detach().requires_grad_()
        (grad,) = torch.autograd.grad(topk_distillation(x, ids, teacher), x, w)
        check(want_loss, grad, logits, ids, teacher, w, 1.0)
        loss, grad = topk_distillation_loss_and_grad(view, ids, teacher, w, out=view)   # last: overwrites the logits
        check(loss, grad, logits, ids, teacher, w, 1.0)
        rest = store.clone()
        rest[first:first + T * pitch].view(T, pitch)[:, :V] = 5.0
        assert rest.eq(5).all()                                                            # nothing between the rows
    t_wide = torch.full((T, K + 3), 9.0, device="cuda")
    t_wide[:, 2:2 + K] = teacher
    i_wide = torch.zeros(T, K + 1, dtype=torch.int32, device="cuda")
    i_wide[:, 1:] = ids
    loss, grad = topk_distillation_loss_and_grad(logits, i_wide[:, 1:], t_wide[:, 2:2 + K], w)
    assert torch.equal(loss, want_loss) and torch.equal(grad, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 600001), (torch.float32, 300001)])
def test_rows_longer_than_a_cluster_holds(dtype, V):
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad
    from steptronoss_b200.ops.distillation import _fits_row

    assert not _fits_row(V, dtype.itemsize) and _fits_row(V // 2, dtype.itemsize)
    logits, ids, teacher, w = make(2, V, 30, seed=5, dtype=dtype, device="cuda")
    ids[0, 3] = ids[0, 2]
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w, 0.7)
    # this kernel adds V / 512 exponentials per thread: a longer chain than the bound's 200, of V / 512 + 16
    assert V / 512 + 16 < 1200
    want, wgrad, p, q = oracle(logits, ids, teacher, 0.7, weights=w)
    loss_tol, grad_tol = bounds(logits.cpu(), teacher.cpu(), 0.7, p, q, wgrad, w.double().cpu(), dtype)
    more = 1000 * 2.0 ** -24
    assert (loss.double().cpu() - want).abs().max() <= loss_tol + more
    assert ((grad.double().cpu() - wgrad).abs() <= grad_tol + w.double().cpu()[:, None] / 0.7 * p * more).all()
    buf = logits.clone()
    loss2, _ = topk_distillation_loss_and_grad(buf, ids, teacher, w, 0.7, out=buf)
    assert torch.equal(loss, loss2) and torch.equal(buf, grad)
    x = logits.clone().requires_grad_()
    tok = topk_distillation(x, ids, teacher, 0.7)
    assert torch.equal(tok.detach(), loss)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_longest_row_of_the_one_pass_kernel_with_the_most_entries(dtype):
    from steptronoss_b200.ops import native, topk_distillation_loss_and_grad

    V = native.load().stb_distill_row_limit(dtype.itemsize)
    logits, ids, teacher, w = make(1, V, 1024, seed=10, dtype=dtype, device="cuda")
    ids[0, 3], ids[0, 4] = V - 1, 0
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    torch.cuda.synchronize()
    native.raise_if_kernel_error()
    check(loss, grad, logits, ids, teacher, w, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V,K", [(torch.bfloat16, 400001, 1024), (torch.bfloat16, 585000, 1024), (torch.float32, 290001, 40)])
def test_many_long_rows(dtype, V, K):
    """One CTA per row as long as its bitmaps leave room for a ring, and the kernel behind it."""
    from steptronoss_b200.ops import native, topk_distillation

    T, rows = 300, [0, 150, 299]
    logits, ids, teacher, w = make(len(rows), V, K, seed=13, dtype=dtype, device="cuda")
    ids[1, 5], ids[1, 6], ids[2, 0] = 7, 7, V - 1
    all_x = torch.zeros(T, V, dtype=dtype, device="cuda")
    all_x[rows] = logits
    all_ids, all_t, all_w = ids.repeat(100, 1), teacher.repeat(100, 1), torch.ones(T, device="cuda")
    all_ids[rows], all_t[rows], all_w[rows] = ids, teacher, w
    tok = topk_distillation(all_x.requires_grad_(), all_ids, all_t)
    (grad,) = torch.autograd.grad(tok, all_x, all_w)
    torch.cuda.synchronize()
    native.raise_if_kernel_error()
    want, wgrad, p, q = oracle(logits, ids, teacher, 1.0, weights=w)
    loss_tol, grad_tol = bounds(logits.cpu(), teacher.cpu(), 1.0, p, q, wgrad, w.double().cpu(), dtype)
    # one CTA adds V / 1024 exponentials into each of a thread's four sums, 572 at most: 400 more than the bound's 200
    more = 400 * 2.0 ** -24
    assert (tok.detach()[rows].double().cpu() - want).abs().max() <= loss_tol + more
    assert ((grad[rows].double().cpu() - wgrad).abs() <= grad_tol + w.double().cpu()[:, None] * p * more).all()


@pytest.mark.gpu
def test_more_elements_than_32_bits_count():
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    T, V, K, last = 14200, 151936, 8, 3
    assert T * V > 2 ** 31
    tail, ids, teacher, w = make(last, V, K, seed=11, dtype=torch.bfloat16, device="cuda")
    logits = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    logits[-last:] = tail
    all_ids = torch.zeros(T, K, dtype=torch.int64, device="cuda")
    all_t = torch.full((T, K), -INF, device="cuda")
    all_w = torch.ones(T, device="cuda")
    all_ids[-last:], all_t[-last:], all_w[-last:] = ids, teacher, w
    alone = topk_distillation(logits.requires_grad_(), all_ids, all_t)
    (grad,) = torch.autograd.grad(alone, logits, all_w)
    assert alone[:-last].eq(0).all() and not grad[:-last].any()
    check(alone.detach()[-last:], grad[-last:], tail, ids, teacher, w, 1.0)
    del grad
    logits = logits.detach()
    loss, grad = topk_distillation_loss_and_grad(logits, all_ids, all_t, all_w, out=logits)
    assert loss[:-last].eq(0).all() and not grad[:-last].any()
    check(loss[-last:], grad[-last:], tail, ids, teacher, w, 1.0)


@pytest.mark.gpu
def test_many_entries():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(3, 1500, 1024, device="cuda")
    ids[1] = ids[1] % 40                            # every id about 25 times
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    check(loss, grad, logits, ids, teacher, w, 1.0)
    loss, grad = topk_distillation_loss_and_grad(logits, ids[:, :0], teacher[:, :0], w)
    assert loss.eq(0).all() and grad.eq(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shards_joined_by_hand_equal_the_whole(dtype):
    """The kernels of a sharded vocabulary, the all-reduces done on one device."""
    from steptronoss_b200.ops import distillation as d
    from steptronoss_b200.ops import native

    T, V, K, tau, parts = 5, 3000, 21, 2.0, 3
    logits, ids, teacher, w = make(T, V, K, seed=6, dtype=dtype, device="cuda")
    ids[0, 0] = V + 5
    teacher[1] = -INF
    logits[2, :1000] = -INF                        # one shard without any probability
    ids[2] = torch.arange(1500, 1500 + K, device="cuda")
    lib, st = native.load(), native.stream()
    stats, picked = [], []
    for r in range(parts):
        x = logits[:, r * 1000:(r + 1) * 1000]
        s = torch.empty(T, 4, device="cuda")
        pk = torch.empty(T, K, device="cuda")
        assert lib.stb_distill_stats(x.data_ptr(), x.stride(0), ids.data_ptr(), 1, ids.stride(0), teacher.data_ptr(), K,
                                     s.data_ptr(), pk.data_ptr(), T, 1000, K, r * 1000, V, 1 / tau, x.element_size(), st) == 0
        stats.append(s)
        picked.append(pk)
    top = torch.stack([s[:, 0] for s in stats]).amax(0)
    whole = stats[0].clone()
    whole[:, 1] = sum(torch.where(s[:, 0] == -INF, s[:, 1], s[:, 1] * torch.exp2(s[:, 0] - top)) for s in stats)
    whole[:, 0] = top
    together = sum(picked)
    loss = torch.empty(T, device="cuda")
    assert lib.stb_distill_loss(ids.data_ptr(), 1, ids.stride(0), teacher.data_ptr(), K, whole.data_ptr(),
                                together.data_ptr(), loss.data_ptr(), T, K, V, 1 / tau, st) == 0
    grad = torch.empty_like(logits)
    for r in range(parts):
        sl = slice(r * 1000, (r + 1) * 1000)
        d._grad_kernel(logits[:, sl], ids, teacher, tau, w, whole, grad[:, sl], r * 1000, V)
    check(loss, grad, logits, ids, teacher, w, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,chunk", [(5, 64, 1000, 2048), (300, 128, 5000, 128), (257, 256, 151936, 100)])
def test_fused_head_follows_the_definition(T, H, V, chunk):
    from steptronoss_b200.ops import fused_linear_topk_distillation, native

    torch.manual_seed(0)
    K, tau = 16, 2.0
    _, ids, teacher, w = make(T, V, K, seed=7, device="cuda")
    teacher[1] = -INF
    w[2] = 0.0
    h = torch.randn(T, H, device="cuda").to(torch.bfloat16).requires_grad_()
    head = (torch.randn(V, H, device="cuda") * 3 / H ** 0.5).to(torch.bfloat16).requires_grad_()
    total, tok = fused_linear_topk_distillation(h, head, ids, teacher, w, tau, chunk_tokens=chunk)
    dh, dw = torch.autograd.grad(total, [h, head], retain_graph=True)
    dh2, _ = torch.autograd.grad(total, [h, head], torch.tensor(0.5, device="cuda"))
    torch.cuda.synchronize()
    native.raise_if_kernel_error()
    logits = h.detach().double() @ head.detach().double().t()
    want, g, p, q = oracle(logits, ids, teacher, tau, weights=w)
    # the logits are sums of H products of size 3 sqrt(H) / sqrt(H) in fp32: H roundings of 2^-24 of sum |a b| at most
    mag = float((h.detach().double().abs() @ head.detach().double().abs().t()).max())
    e = H * 2.0 ** -24 * mag / tau
    loss_tol, _ = bounds(logits.cpu(), teacher.cpu(), tau, p, q, g, w.double().cpu(), torch.bfloat16)
    assert (tok.double().cpu() - want).abs().max() <= loss_tol + 2 * e
    assert abs(float(total.detach()) - float((want * w.double().cpu()).sum())) <= (loss_tol + 2 * e) * float(w.sum()) * 1.01
    # gradient rows are rounded to bf16 (2^-8 of each), the products summed in fp32 and rounded once more
    for got, a, b in ((dh, g, head.detach().double().cpu()), (dw, g.t(), h.detach().double().cpu())):
        exact, size = a @ b, a.abs() @ b.abs()
        tol = size * (2.0 ** -8 + 2 * e + 1e-4) + exact.abs() * 2.0 ** -8 + 1e-30
        assert ((got.double().cpu() - exact).abs() <= tol).all()
    assert torch.allclose(dh2.float(), 0.5 * dh.float(), rtol=2.0 ** -8, atol=0)
    with torch.no_grad():
        total2, tok2 = fused_linear_topk_distillation(h, head, ids, teacher, w, tau, chunk_tokens=chunk)
    assert torch.equal(tok, tok2) and total2 == total


@pytest.mark.gpu
def test_fused_head_without_tokens():
    from steptronoss_b200.ops import fused_linear_topk_distillation

    _, ids, teacher, w = make(3, 64, 2, device="cuda")
    h = torch.zeros(0, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    head = torch.zeros(64, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    total, tok = fused_linear_topk_distillation(h, head, ids[:0], teacher[:0], w[:0])
    dh, dw = torch.autograd.grad(total, [h, head])
    assert total == 0 and tok.shape == (0,) and dh.shape == (0, 16) and dw.eq(0).all()


@pytest.mark.gpu
def test_fused_head_adds_into_main_grad():
    from steptronoss_b200.ops import fused_linear_topk_distillation

    torch.manual_seed(0)
    T, H, V, K = 90, 64, 512, 8
    _, ids, teacher, w = make(T, V, K, seed=8, device="cuda")
    h = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    head = torch.nn.Parameter((torch.randn(V, H, device="cuda") * 0.3).to(torch.bfloat16))
    total, _ = fused_linear_topk_distillation(h, head, ids, teacher, w, chunk_tokens=32)
    total.backward()
    plain = head.grad.float().clone()
    head.grad, head.main_grad = None, torch.ones(V, H, device="cuda")
    total, _ = fused_linear_topk_distillation(h, head, ids, teacher, w, chunk_tokens=32)
    total.backward()
    assert head.grad is None and head.grad_added_to_main_grad
    assert torch.allclose(head.main_grad - 1, plain, rtol=2.0 ** -8, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_fused_head_leaves_main_grad_alone_without_gradients(mode):
    from steptronoss_b200.ops import fused_linear_topk_distillation

    torch.manual_seed(0)
    T, H, V, K = 40, 64, 512, 8
    _, ids, teacher, w = make(T, V, K, seed=9, device="cuda")
    h = torch.randn(T, H, device="cuda").to(torch.bfloat16).requires_grad_()
    head = torch.nn.Parameter((torch.randn(V, H, device="cuda") * 0.3).to(torch.bfloat16))
    head.main_grad = torch.ones(V, H, device="cuda")
    with mode():
        total, tok = fused_linear_topk_distillation(h, head, ids, teacher, w, chunk_tokens=32)
    assert head.main_grad.eq(1).all() and not total.requires_grad and not hasattr(head, "grad_added_to_main_grad")
    # with gradients the same loss, and then they are there
    total2, tok2 = fused_linear_topk_distillation(h, head, ids, teacher, w, chunk_tokens=32)
    assert torch.equal(tok, tok2) and total == total2 and head.main_grad.ne(1).any()


@pytest.mark.gpu
def test_gradient_agrees_with_differences_on_the_gpu():
    from steptronoss_b200.ops import topk_distillation

    T, V, K, tau, h = 5, 400, 7, 1.5, 0.02
    logits, ids, teacher, w = make(T, V, K, seed=12, device="cuda")
    ids[0, 1] = ids[0, 0]
    d = torch.randint(0, 2, (T, V), device="cuda").float() * 2 - 1
    x = logits.clone().requires_grad_()
    (grad,) = torch.autograd.grad(topk_distillation(x, ids, teacher, tau), x, torch.ones(T, device="cuda"))
    slope = (topk_distillation(logits + h * d, ids, teacher, tau) - topk_distillation(logits - h * d, ids, teacher, tau)) / (2 * h)
    _, wgrad, p, q = oracle(logits, ids, teacher, tau)
    loss_tol, _ = bounds(logits.cpu(), teacher.cpu(), tau, p, q, wgrad, torch.ones(T, dtype=torch.float64), torch.float32)
    # the loss is off by loss_tol on either side; along d = +-1 its third derivative is a third central moment of values in
    # [-1, 1] over tau^3, at most 2 / tau^3; logits +- h d are rounded by 2^-24 of 15 at most, times a gradient of size 1
    tol = loss_tol / h + h * h / 6 * 2 / tau ** 3 + 15 * 2.0 ** -24 / h + 1e-5
    assert ((grad * d).sum(1).double() - slope.double()).abs().max() <= tol
    # and that says something: logits of spread 30 at most give A <= 1.4427 * 30 / 1.5 + 20 = 49, so that loss_tol / h is at
    # most (4 * 49 + 212 + 2 * 49 * (2 * 49 + 48)) 2^-24 / 0.02 = 0.044, the other terms 2e-4; the slopes are about 0.4
    assert tol < 0.05


@pytest.mark.gpu
def test_kernels_on_a_side_stream_and_in_a_graph():
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    logits, ids, teacher, w = make(17, 30000, 24, dtype=torch.bfloat16, device="cuda")
    want_loss, want = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, want_loss) and torch.equal(grad, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    logits.mul_(0.5)
    want_loss, want = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and torch.equal(grad, want)


@pytest.mark.gpu
def test_gpu_refusals():
    from steptronoss_b200.ops import fused_linear_topk_distillation, topk_distillation

    _, ids, teacher, w = make(4, 16, 2, device="cuda")
    with pytest.raises(TypeError):
        topk_distillation(torch.zeros(4, 16, dtype=torch.float16, device="cuda"), ids, teacher)
    with pytest.raises(ValueError):
        topk_distillation(torch.zeros(4, 16, device="cuda"), ids.cpu(), teacher)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        fused_linear_topk_distillation(bf(4, 8).float(), bf(16, 8), ids, teacher, w)
    with pytest.raises(ValueError):
        fused_linear_topk_distillation(bf(4, 8), bf(17, 8), ids, teacher, w)
    with pytest.raises(ValueError):
        fused_linear_topk_distillation(bf(4, 12), bf(16, 12), ids, teacher, w)


def lowest_rows(T, V, K, dtype, device, tau):
    """Rows masked with the type's lowest value: in part, an entry among it; throughout; throughout but for -inf; a logit of
    the type's largest value; entries of a teacher that is masked so; and ordinary rows behind them."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits, ids, teacher, w = make(T, V, K, seed=20, dtype=dtype)
    ids[:, 0] = torch.arange(T) % V
    for j in range(1, K):                           # distinct ids
        ids[:, j] = (ids[:, 0] + 1 + 3 * j) % V
    logits[0, V // 2:] = low
    logits[0, ids[0, 1]] = low
    logits[1] = low
    logits[2] = low
    logits[2, V // 3:V // 2] = -INF
    ids[2] = torch.arange(K)
    logits[3, ids[3, 2]] = high
    teacher[4, 1:] = torch.finfo(torch.float32).min
    logits[5, ids[5]] = 0.75 * low                  # all entries masked
    want, wgrad, p, q = oracle(logits, ids, teacher, tau, weights=w)
    usual = torch.where(logits.abs() > 1e38, 0.0, logits.float())
    usual_t = torch.where(teacher < -1e38, 0.0, teacher)
    # logits of that size leave p = 0 or equal parts: exponents are 0 or far below the range.  The other terms are those of
    # `bounds`; a loss of that size is q times a difference, off by less than loss_tol of itself
    loss_tol, grad_tol = bounds(usual, usual_t, tau, p, q, wgrad, w.double(), dtype)
    big = torch.finfo(torch.float32).max
    assert ((want - big).abs() > 1e-3 * big).all()

    def verify(loss, grad):
        loss = loss.double().cpu()
        assert loss[want > big].eq(INF).all()
        fine = want < big
        assert ((loss - want)[fine].abs() <= loss_tol * (1 + want[fine].abs())).all(), (loss[:6], want[:6])
        assert ((grad.double().cpu() - wgrad).abs() <= grad_tol).all()

    return [t.to(device) for t in (logits, ids, teacher, w)], verify


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("T,V,K", [(6, 40, 3), (7, 5003, 12)])
def test_logits_masked_with_the_lowest_value(device, dtype, tau, T, V, K):
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    (logits, ids, teacher, w), verify = lowest_rows(T, V, K, dtype, device, tau)
    verify(*topk_distillation_loss_and_grad(logits, ids, teacher, w, tau))
    x = logits.clone().requires_grad_()
    tok = topk_distillation(x, ids, teacher, tau)
    verify(tok.detach(), torch.autograd.grad(tok, x, w)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,V", [(torch.bfloat16, 310, 3001), (torch.float32, 310, 3001),     # one CTA per row
                                       (torch.bfloat16, 6, 151936), (torch.float32, 6, 151936),     # clusters
                                       (torch.bfloat16, 6, 600001), (torch.float32, 6, 300001)])    # three kernels
def test_logits_masked_with_the_lowest_value_in_every_kernel(dtype, T, V):
    from steptronoss_b200.ops import native, topk_distillation, topk_distillation_loss_and_grad

    (logits, ids, teacher, w), verify = lowest_rows(T, V, 9, dtype, "cuda", 1.0)
    verify(*topk_distillation_loss_and_grad(logits, ids, teacher, w))
    x = logits.clone().requires_grad_()
    tok = topk_distillation(x, ids, teacher)
    verify(tok.detach(), torch.autograd.grad(tok, x, w)[0])
    torch.cuda.synchronize()
    native.raise_if_kernel_error()


def test_statistics_of_large_rows_are_joined():
    """Rows by what their two shards hold: (top, sum), for large rows (max, -count)."""
    from steptronoss_b200.ops.distillation import _shard_keys, _shard_sums

    low, cases = -3.4e38, []
    cases.append(((5.0, 2.0), (3.0, 4.0), (5.0, 3.0)))                  # ordinary: 2 + 4 / 4
    cases.append(((-INF, 0.0), (3.0, 4.0), (3.0, 4.0)))
    cases.append(((-INF, 0.0), (-INF, 0.0), (-INF, 0.0)))
    cases.append(((low, -7.0), (3.0, 4.0), (3.0, 4.0)))                 # masked beside ordinary
    cases.append(((low, -7.0), (-2e9, 4.0), (-2e9, 4.0)))
    cases.append(((low, -7.0), (low, -2.0), (low, -9.0)))               # masked throughout
    cases.append(((low, -7.0), (-2.4e38, -2.0), (-2.4e38, -2.0)))
    cases.append(((low, -7.0), (-INF, 0.0), (low, -7.0)))
    cases.append(((3e38, -1.0), (9.0, 4.0), (3e38, -1.0)))
    cases.append(((3e38, -1.0), (low, -4.0), (3e38, -1.0)))
    cases.append(((3e38, -1.0), (9.0, math.nan), (3e38, math.nan)))     # a NaN stays visible
    a, b, want = (torch.tensor([c[i] for c in cases]) for i in range(3))
    keys = torch.maximum(_shard_keys(a), _shard_keys(b))
    (sa, large), (sb, other) = _shard_sums(a, keys), _shard_sums(b, keys)
    assert torch.equal(large, other) and torch.equal(large, want[:, 1].lt(0) | want[:, 1].isnan())
    assert torch.equal(torch.where(large, keys[1], keys[0]), want[:, 0])
    got = torch.where(large, -(sa + sb), sa + sb)
    assert torch.allclose(got, want[:, 1], rtol=0, atol=0, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [1, 3])
def test_shards_with_the_lowest_value_equal_the_whole(dtype, parts):
    """The kernels of a sharded vocabulary on logits masked with the type's lowest value."""
    from steptronoss_b200.ops import distillation as d
    from steptronoss_b200.ops import native

    T, V, K, tau = 7, 3000, 9, 0.5
    (logits, ids, teacher, w), verify = lowest_rows(T, V, K, dtype, "cuda", tau)
    lib, st, width = native.load(), native.stream(), V // parts
    stats, picked = [], []
    for r in range(parts):
        x = logits[:, r * width:(r + 1) * width]
        stats.append(torch.empty(T, 4, device="cuda"))
        picked.append(torch.empty(T, K, device="cuda"))
        assert lib.stb_distill_stats(x.data_ptr(), x.stride(0), ids.data_ptr(), 1, ids.stride(0), teacher.data_ptr(), K,
                                     stats[r].data_ptr(), picked[r].data_ptr(), T, width, K, r * width, V, 1 / tau,
                                     x.element_size(), st) == 0
    keys = torch.stack([d._shard_keys(s) for s in stats]).amax(0)
    sums = sum(d._shard_sums(s, keys)[0] for s in stats)
    large = d._shard_sums(stats[0], keys)[1]
    whole = stats[0].clone()
    whole[:, 0], whole[:, 1] = torch.where(large, keys[1], keys[0]), torch.where(large, -sums, sums)
    together, loss, grad = sum(picked), torch.empty(T, device="cuda"), torch.empty_like(logits)
    assert lib.stb_distill_loss(ids.data_ptr(), 1, ids.stride(0), teacher.data_ptr(), K, whole.data_ptr(),
                                together.data_ptr(), loss.data_ptr(), T, K, V, 1 / tau, st) == 0
    for r in range(parts):
        sl = slice(r * width, (r + 1) * width)
        d._grad_kernel(logits[:, sl], ids, teacher, tau, w, whole, grad[:, sl], r * width, V)
    verify(loss, grad)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 3e9, 1e12, 1e30])
def test_logits_of_any_size(device, size):
    """Rows whose numbers all lie near `size`, a few units in the last place apart, on both sides of zero."""
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    T, V, K = 4, 700, 5
    g = torch.Generator().manual_seed(23)
    base = torch.tensor([size, -size, size, -size])[:, None].expand(T, V).contiguous()
    logits = base.view(torch.int32).add(torch.randint(0, 4, (T, V), generator=g, dtype=torch.int32)).view(torch.float32)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)])
    teacher, w = torch.randn(T, K, generator=g), torch.ones(T)
    for tau in (0.25, 1.0, 3.0):
        loss, grad = topk_distillation_loss_and_grad(*(t.to(device) for t in (logits, ids, teacher, w)), tau)
        want, wgrad, p, q = oracle(logits, ids, teacher, tau)
        # only differences from the maximum count, and they are exact; the rounding of c * max s, half a unit in its last
        # place, cancels, but passes through one sum and one logarithm of its size
        near = logits - logits.amax(1, keepdim=True)
        loss_tol, grad_tol = bounds(near, teacher, tau, p, q, wgrad, w.double(), torch.float32)
        more = 4 * min(1.4427 * size / tau, 2.0 ** 31) * 2.0 ** -48
        assert ((loss.double().cpu() - want).abs() <= loss_tol * (1 + want) + more).all()
        # beside large maxima what lies 64 or more below in the exponent may count as nothing
        assert ((grad.double().cpu() - wgrad).abs() <= grad_tol + (p * more + 2.0 ** -64) / tau).all()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["one element off", "single token from an odd pitch", "single token one element off",
                                 "one row repeated", "rows that overlap", "odd pitch"])
def test_fused_head_takes_hidden_states_on_any_address(how):
    """The same numbers whatever the layout: the fp32 logits of the framework's own product."""
    from steptronoss_b200.ops import fused_linear_topk_distillation

    torch.manual_seed(0)
    T, H, V, K = 90, 64, 1000, 8
    if "single" in how:
        T = 1
    _, ids, teacher, w = make(T, V, K, seed=21, device="cuda")
    store = torch.randn(T * (H + 3) + 1, device="cuda").to(torch.bfloat16)
    h = {"one element off": lambda: store[1:1 + T * H].view(T, H),
         "single token from an odd pitch": lambda: store[:H + 3].view(1, H + 3)[:, :H],
         "single token one element off": lambda: store[1:1 + H].view(1, H),
         "one row repeated": lambda: store[:H].expand(T, H),
         "rows that overlap": lambda: store.as_strided((T, H), (8, 1)),
         "odd pitch": lambda: store[:T * (H + 3)].view(T, H + 3)[:, :H]}[how]()
    head = (torch.randn(V, H, device="cuda") * 0.8).to(torch.bfloat16).requires_grad_()

    def run(x):
        total, tok = fused_linear_topk_distillation(x, head, ids, teacher, w, chunk_tokens=32)
        return (total.detach(), tok, *torch.autograd.grad(total, [x, head]))

    want = run(torch.empty(T, H, dtype=h.dtype, device="cuda").copy_(h).requires_grad_())
    for a, b in zip(run(h.detach().requires_grad_()), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_fused_head_takes_a_main_grad_on_any_address():
    from steptronoss_b200.ops import fused_linear_topk_distillation

    torch.manual_seed(0)
    T, H, V, K = 90, 64, 512, 8
    _, ids, teacher, w = make(T, V, K, seed=8, device="cuda")
    h = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    head = torch.nn.Parameter((torch.randn(V, H, device="cuda") * 0.3).to(torch.bfloat16))

    def run(main_grad):
        head.main_grad = main_grad.fill_(1.0)
        total, _ = fused_linear_topk_distillation(h, head, ids, teacher, w, chunk_tokens=32)
        total.backward()
        assert head.grad is None
        return head.main_grad

    want = run(torch.empty(V, H, device="cuda"))
    got = run(torch.empty(V * H + 1, device="cuda")[1:].view(V, H))
    # three blocks and the 1 that was there, in another order: four roundings of 2^-24 on each side
    assert ((got - want).abs() <= 8 * 2.0 ** -24 * (1 + (want - 1).abs() * 3)).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("main_grad", [False, True])
def test_fused_head_passes_over_hidden_states_that_do_not_count(device, main_grad):
    """Tokens of weight 0 and without entries may hold anything, in their hidden states too."""
    from steptronoss_b200.ops import fused_linear_topk_distillation

    torch.manual_seed(0)
    T, H, V, K = 70, 32, 200, 5
    _, ids, teacher, w = make(T, V, K, seed=22)
    teacher[3], teacher[40], ids[69] = -INF, -INF, V
    w[2], w[33] = 0.0, 0.0
    dead = torch.tensor([2, 3, 33, 40, 69])
    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    ids, teacher, w, h = ids.to(device), teacher.to(device), w.to(device), torch.randn(T, H).to(device, dtype)
    head = torch.nn.Parameter((torch.randn(V, H) * 0.5).to(device, dtype))

    def run(x):
        x = x.clone().requires_grad_()
        head.grad = None
        if main_grad and device == "cuda":
            head.main_grad = torch.zeros(V, H, device="cuda")
        total, tok = fused_linear_topk_distillation(x, head, ids, teacher, w, 2.0, chunk_tokens=32)
        total.backward()
        return total.detach(), tok, x.grad, head.main_grad if main_grad and device == "cuda" else head.grad

    h[dead] = 0
    want = run(h)
    h[dead] = torch.tensor([math.nan, INF, -INF, math.nan, math.nan], dtype=dtype, device=device)[:, None]
    total, tok, dh, dw = run(h)
    assert total == want[0] and torch.equal(dw, want[3]) and torch.equal(dh, want[2]) and dh[dead].eq(0).all()
    live = torch.ones(T, dtype=torch.bool)
    live[dead] = False
    assert torch.equal(tok[live], want[1][live]) and tok[[3, 40, 69]].eq(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,T,V,K", [(torch.bfloat16, 8, 151936, 1024), (torch.float32, 300, 151936, 200),
                                         (torch.bfloat16, 700, 50257, 200)])
def test_the_gradient_over_the_logits_waits_for_every_reader(dtype, T, V, K):
    """The first CTA of a cluster reads the logits at all entries, wherever they lie, before others write over them."""
    from steptronoss_b200.ops import topk_distillation_loss_and_grad

    g = torch.Generator(device="cuda").manual_seed(24)
    logits = (torch.randn(T, V, device="cuda", generator=g) * 3).to(dtype)
    step = V // K
    ids = torch.arange(K, device="cuda") * step + torch.randint(0, step, (T, K), device="cuda", generator=g)
    teacher, w = torch.randn(T, K, device="cuda", generator=g), torch.rand(T, device="cuda", generator=g)
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    buf = torch.empty_like(logits)
    for _ in range(20):
        buf.copy_(logits)
        again, _ = topk_distillation_loss_and_grad(buf, ids, teacher, w, out=buf)
        assert torch.equal(again, loss) and torch.equal(buf, grad)


@pytest.mark.parametrize("rows, vocab", [(2 ** 28, 1), (2 ** 31 + 1, 1), (2 ** 32 + 3, 1), (1, 2 ** 30 + 1), (1, 2 ** 32 + 3)])
def test_sizes_beyond_the_kernels_are_refused(rows, vocab):
    """Sizes cross the C interface as 32-bit numbers: larger ones would be taken for smaller ones there."""
    from steptronoss_b200.ops import topk_distillation, topk_distillation_loss_and_grad

    logits = torch.zeros(1, 1).expand(rows, vocab)
    ids, teacher = torch.zeros(1, 1, dtype=torch.long).expand(rows, 1), torch.zeros(1, 1).expand(rows, 1)
    with pytest.raises(ValueError, match="at most"):
        topk_distillation(logits, ids, teacher)
    with pytest.raises(ValueError, match="at most"):
        topk_distillation_loss_and_grad(logits, ids, teacher, torch.zeros(1).expand(rows))


def test_fused_head_refuses_sizes_beyond_the_kernels():
    from steptronoss_b200.ops import fused_linear_topk_distillation as f

    for rows, vocab in ((2 ** 31 + 8, 8), (1, 2 ** 32 + 8)):
        ids, teacher = torch.zeros(1, 1, dtype=torch.long).expand(rows, 1), torch.zeros(1, 1).expand(rows, 1)
        with pytest.raises(ValueError, match="at most"):
            f(torch.zeros(1, 8).expand(rows, 8), torch.zeros(1, 8).expand(vocab, 8), ids, teacher, torch.zeros(1).expand(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(6, 151936), (300, 50257)])
def test_large_rows_are_looked_at_again_before_they_are_overwritten(dtype, T, V):
    from steptronoss_b200.ops import native, topk_distillation_loss_and_grad

    (logits, ids, teacher, w), verify = lowest_rows(T, V, 9, dtype, "cuda", 1.0)
    loss, grad = topk_distillation_loss_and_grad(logits, ids, teacher, w)
    verify(loss, grad)
    buf = torch.empty_like(logits)
    for _ in range(10):
        buf.copy_(logits)
        again, _ = topk_distillation_loss_and_grad(buf, ids, teacher, w, out=buf)
        assert torch.equal(again, loss) and torch.equal(buf, grad)
    torch.cuda.synchronize()
    native.raise_if_kernel_error()


def _join_worker(rank, world, port, q):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1",
                      MASTER_PORT=str(port))
    torch.set_num_threads(1)
    try:
        import torch.distributed as dist

        from steptronoss_b200.ops.distillation import _join_shards

        dist.init_process_group("gloo", rank=rank, world_size=world)
        shard = [[(5.0, 2.0), (-3.4e38, -7.0), (-3.4e38, -7.0), (-INF, 0.0)],
                 [(3.0, 4.0), (3.0, 4.0), (-3.4e38, -2.0), (9.0, 1.5)]][rank]
        stats = torch.tensor([(*pair, 1.0, 2.0) for pair in shard])
        picked = torch.full((4, 3), float(rank))
        _join_shards(stats, picked, dist.group.WORLD)
        q.put((rank, stats.tolist(), picked.tolist(), None))
        dist.barrier()
        dist.destroy_process_group()
    except BaseException:
        import traceback

        q.put((rank, None, None, traceback.format_exc()))
        raise


def test_shards_are_joined_over_a_group():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = free_port()
    procs = [ctx.Process(target=_join_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        for _ in range(2):
            _, stats, picked, err = q.get(timeout=120)
            assert err is None, err
            want = torch.tensor([(5.0, 3.0, 1.0, 2.0), (3.0, 4.0, 1.0, 2.0), (-3.4e38, -9.0, 1.0, 2.0), (9.0, 1.5, 1.0, 2.0)])
            assert torch.equal(torch.tensor(stats), want) and torch.tensor(picked).eq(1).all()
    finally:
        for p in procs:
            p.join(timeout=30)
            if p.is_alive():
                p.kill()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_fused_head_refuses_a_main_grad_that_does_not_fit(device):
    """The weight gradient's product goes by the shape of w: it would write behind a smaller main_grad."""
    from steptronoss_b200.ops import fused_linear_topk_distillation as f

    dtype = torch.bfloat16 if device == "cuda" else torch.float32
    ids, t, w = torch.zeros(4, 2, dtype=torch.long, device=device), torch.zeros(4, 2, device=device), torch.ones(4, device=device)
    h, head = torch.zeros(4, 8, device=device, dtype=dtype), torch.nn.Parameter(torch.zeros(16, 8, device=device, dtype=dtype))
    for bad in (torch.zeros(8, 8, device=device), torch.zeros(128, device=device), torch.zeros(16, 16, device=device),
                torch.zeros(16, 8, device=device, dtype=torch.float16), torch.zeros(16, 8, device="meta")):
        head.main_grad = bad
        with pytest.raises(ValueError, match="main_grad"):
            f(h, head, ids, t, w)
    head.main_grad = torch.zeros(16, 8, device=device)
    f(h, head, ids, t, w)
    for empty in (torch.zeros(0, 8, device=device, dtype=dtype), torch.zeros(16, 0, device=device, dtype=dtype)):
        with pytest.raises(ValueError, match="vocabulary"):
            f(h[:, :empty.shape[1]], empty, ids, t, w)
