"""topk_distillation against the definition in 64 bits, and what it refuses."""
import pytest
import torch

import tilelang_ascend_b200 as dsa

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
INF = float("inf")


def definition(student, teacher, indices, kind, over, T, grad):
    """Losses and student gradients of rows [R, V] in 64 bits, and the sizes their error bounds are made of."""
    R, V = student.shape
    loss, d = torch.zeros(R, dtype=torch.float64), torch.zeros(R, V, dtype=torch.float64)
    slack, d_slack = torch.zeros(R, dtype=torch.float64), torch.zeros(R, V, dtype=torch.float64)
    for r in range(R):
        cols = torch.arange(V) if indices is None else indices[r].long()
        there = (cols >= 0) & (cols < V)
        there &= ~(student[r, cols.clamp(0, V - 1)].double() == -INF)
        cols, t = cols[there], teacher[r][there].double()
        z = student[r].double() / T
        w = torch.exp((t - t.max()) / T) if kind == "logits" and t.numel() and t.max() > -INF else (t.clamp(min=0) if kind == "weights" else t * 0)
        if not cols.numel() or float(w.nan_to_num(0).sum()) == 0:
            continue
        p = w / w.sum()
        base = z if over == "row" else z[cols]
        m, logz = base.max(), torch.logsumexp(base, 0)
        log_s = z[cols] - logz
        terms = torch.where(p > 0, p * (torch.log(p) - log_s), torch.zeros_like(p))
        loss[r] = terms.sum()
        soft = torch.exp(base - logz)
        g = grad[r].double() / T
        if over == "row":
            d[r] = g * soft
        else:
            d[r].index_add_(0, cols, g * soft)
        d[r].index_add_(0, cols, -g * p)
        # fp32: exp((x - m) / T) is off by 2^-22 and by the rounding of its argument, three steps of |x - m| / T; sums of up to n / 256 + 12
        # additions; a logarithm and three sums in every term
        steps = (base.numel() / 256 + 12 + cols.numel() / 256) * 2.0 ** -24 + 2.0 ** -21
        e_z = steps + float((soft * (m - base).clamp(max=200)).nan_to_num(0).sum()) * 3 * 2.0 ** -24
        lp = torch.where(p > 0, torch.log(p).abs(), torch.zeros_like(p))
        e_t = steps + float((p * lp).sum()) * 6 * 2.0 ** -24
        sizes = torch.where(p > 0, p * (lp + (m - z[cols]) + (logz - m).abs() + 1), torch.zeros_like(p)).sum()
        slack[r] = float(sizes) * (8 * 2.0 ** -24 + e_t) + e_z + e_t
        d_slack[r] = g.abs() * 1e-30
        ds = g.abs() * soft * (e_z + 3 * 2.0 ** -24 * (m - base).clamp(max=200).nan_to_num(0) + 2.0 ** -21)
        dp = g.abs() * p * (e_t + 3 * 2.0 ** -24 * (lp + 20) + 2.0 ** -21)
        if over == "row":
            d_slack[r] += ds
        else:
            d_slack[r].index_add_(0, cols, ds)
        d_slack[r].index_add_(0, cols, dp)
    return loss, d, slack, d_slack


def check(student, teacher, indices, kind, over, T, grad=None, dev_student=None):
    R, V = student.shape
    grad = torch.rand(R) + 0.1 if grad is None else grad
    loss, d, slack, d_slack = definition(student, teacher, indices, kind, over, T, grad)
    leaf = (student.cuda() if dev_student is None else dev_student).detach().requires_grad_()
    got = dsa.topk_distillation(leaf, teacher.cuda(), None if indices is None else indices.cuda(), teacher_kind=kind, over=over, temperature=T)
    (dg,) = torch.autograd.grad(got, leaf, grad.cuda())
    got, dg = got.detach().cpu().double(), dg.cpu()
    assert got.shape == (R,) and dg.shape == (R, V) and dg.dtype == student.dtype and dg.is_contiguous()
    assert bool(((got - loss).abs() <= slack + loss.abs() * 2.0 ** -23).all()), f"loss off by {float(((got - loss).abs() - slack).max())}"
    dt = student.dtype
    err, bound = (dg.double() - d).abs(), (d.abs() + d_slack) * HALF_STEP[dt] + d_slack + TINY[dt]
    assert bool((err <= bound).all()), f"gradient off by {float((err - bound).max())}"
    return got, dg


def rows(R, V, K, dtype, kind, seed, listed):
    g = torch.Generator().manual_seed(seed)
    student = (2 * torch.randn((R, V), generator=g)).to(dtype)
    teacher = 2 * torch.randn((R, K), generator=g)
    if kind == "weights":
        teacher = teacher.exp()
    indices = None
    if listed:
        indices = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]).to(torch.int32)
    return g, student, teacher, indices


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["weights", "logits"])
@pytest.mark.parametrize("R,K", [(1, 1), (3, 2), (5, 100), (2, 1025), (2, 4097), (1, 9001)])
def test_lists(R, K, kind, dtype):
    g, student, teacher, _ = rows(R, K, K, dtype, kind, seed=K, listed=False)
    check(student, teacher, None, kind, "list", 1.0)
    check(student, teacher.to(torch.bfloat16), None, kind, "row", 3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,over", [("weights", "list"), ("weights", "row"), ("logits", "row"), ("logits", "list")])
@pytest.mark.parametrize("R,V,K", [(2, 7, 3), (3, 1001, 64), (2, 8193, 2049), (2, 20003, 1), (1, 40000, 8200), (2, 5000, 1024)])
def test_listed_columns(R, V, K, kind, over, dtype):
    g, student, teacher, indices = rows(R, V, K, dtype, kind, seed=V + K, listed=True)
    if K > 2:
        indices[0, 1], indices[-1, 0] = -1, V      # padding, and a column that does not exist
        teacher[0, 1], teacher[-1, 0] = float("nan"), INF
        student[0, indices[0, 2]] = -INF
    check(student, teacher, indices, kind, over, 1.0)
    check(student, teacher.to(torch.float16), indices, kind, over, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("over", ["list", "row"])
def test_masks_that_leave_nothing_and_values_in_masked_places(over, listed):
    V, K = 300, 40 if listed else 300
    for kind in ("weights", "logits"):
        g, student, teacher, indices = rows(8, V, K, torch.float32, kind, seed=1, listed=listed)
        cols = torch.arange(V).repeat(8, 1) if indices is None else indices.long()
        student[0] = -INF                                       # nothing takes part
        teacher[1] = 0.0 if kind == "weights" else -INF         # a teacher that holds nothing
        student[2, cols[2, 3:]] = -INF                          # a few entries left, the teacher's NaN lies among the others
        teacher[2, 3:] = float("nan")
        student[3, cols[3, 1]] = torch.finfo(torch.float32).min / 4   # a finite mask value outside the teacher's support
        teacher[3, 1] = 0.0 if kind == "weights" else -INF
        teacher[4] = teacher[4] * 1e-30 if kind == "weights" else teacher[4] - 1e4
        student[5] += 30000.0                                   # far from zero
        if kind == "weights":
            teacher[6, 0] = -3.0                                # (not below 0: counts as 0)
        if listed:
            indices[7] = -1
        for T in (1.0, 0.25):
            loss, d = check(student, teacher, indices, kind, over, T)
            assert float(loss[0]) == 0 and float(loss[1]) == 0 and not d[:2].any()
            if listed:
                assert float(loss[7]) == 0 and not d[7].any()
    bad = student.clone()
    bad[4, cols[4, 0]] = float("nan")
    loss = dsa.topk_distillation(bad.cuda(), teacher.cuda(), None if indices is None else indices.cuda(), teacher_kind="logits", over=over)
    assert loss.isnan().tolist() == [False] * 4 + [True] + [False] * 3


@pytest.mark.gpu
@pytest.mark.parametrize("over", ["list", "row"])
def test_a_column_listed_twice(over):
    g, student, teacher, indices = rows(4, 500, 20, torch.float32, "weights", seed=4, listed=True)
    indices[:, 7] = indices[:, 3]
    check(student, teacher, indices, "weights", over, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strided_and_unaligned_rows(dtype):
    """Rows of a wider matrix, from an odd column on; lists of two leading dimensions."""
    g, student, teacher, indices = rows(6, 1003, 50, dtype, "logits", seed=2, listed=True)
    wide = torch.zeros((6, 1200), dtype=dtype, device="cuda")
    for first in (1, 4, 8):
        view = wide[:, first:first + 1003]
        view.copy_(student)
        check(student, teacher, indices, "logits", "row", 1.0, dev_student=view)
    loss = dsa.topk_distillation(student.view(2, 3, 1003).cuda(), teacher.view(2, 3, 50).cuda(), indices.view(2, 3, 50).cuda(), teacher_kind="logits", over="row")
    flat = dsa.topk_distillation(student.cuda(), teacher.cuda(), indices.cuda(), teacher_kind="logits", over="row")
    assert loss.shape == (2, 3) and torch.equal(loss.flatten(), flat)
    assert dsa.topk_distillation(student[:0].cuda(), teacher[:0].cuda(), indices[:0].cuda()).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [70001, 65544])
def test_wide_rows_in_several_parts(V, dtype):
    """Rows that several blocks share, in 16-byte units and not, with parts that hold no entry, only masked logits, or the maximum alone."""
    g, student, teacher, indices = rows(4, V, 900, dtype, "logits", seed=V, listed=True)
    indices[1] = indices[1] % 3000                    # all entries in the first part (some columns more than once)
    student[2, 32768:65536] = -INF
    student[3, V - 1] = 40.0
    check(student, teacher, indices, "logits", "row", 2.0)
    check(student, teacher.exp(), indices, "weights", "row", 1.0)


@pytest.mark.gpu
def test_broadcast_rows_and_second_backward():
    g, student, teacher, indices = rows(5, 600, 40, torch.float32, "weights", seed=12, listed=True)
    one = student[:1].cuda().requires_grad_()
    loss = dsa.topk_distillation(one.expand(5, 600), teacher.cuda(), indices.cuda(), over="row")
    (first,) = torch.autograd.grad(loss.sum(), one, retain_graph=True)
    (again,) = torch.autograd.grad(loss.sum(), one)
    _, d, _, slack = definition(student[:1].expand(5, 600), teacher, indices, "weights", "row", 1.0, torch.ones(5))
    assert torch.equal(first, again)
    assert bool(((first[0].cpu().double() - d.sum(0)).abs() <= slack.sum(0) + d.abs().sum(0) * 2.0 ** -22).all())


@pytest.mark.gpu
def test_gradient_by_differences():
    g, student, teacher, indices = rows(1, 60, 9, torch.float32, "weights", seed=6, listed=True)
    _, d = check(student, teacher, indices, "weights", "row", 2.0, grad=torch.ones(1))
    h = 1e-4
    for c in (int(indices[0, 0]), int(indices[0, 8]), 5):
        values = []
        for sign in (1, -1):
            moved = student.double()
            moved[0, c] += sign * h
            values.append(definition(moved, teacher, indices, "weights", "row", 2.0, torch.ones(1))[0])
        want = float((values[0] - values[1]) / (2 * h))
        assert abs(float(d[0, c]) - want) <= 1e-6 + 1e-5 * abs(want)   # (differences: h^2 / 6 times a third derivative below 1)


@pytest.mark.gpu
def test_repeatable_captured_and_on_another_stream():
    g, student, teacher, indices = (t.cuda() if isinstance(t, torch.Tensor) else t for t in rows(40, 9000, 700, torch.float32, "weights", seed=3, listed=True))
    grad = torch.rand(40, device="cuda")

    def step():
        loss, stats = dsa.topk_distillation_raw(student, teacher, indices, over="row")
        return loss, dsa.topk_distillation_bwd_raw(student, teacher, indices, stats, grad, over="row")

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    student.mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other)) and all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.gpu
@pytest.mark.parametrize("V,K,over", [(300, None, "list"), (300, 40, "list"), (300, 40, "row"), (40000, 700, "row")])
def test_a_teacher_whose_sum_is_not_finite(V, K, over):
    """An infinite weight, or weights whose sum fp32 does not hold: NaN in the loss and in the gradient of the entries, other rows as they are."""
    g, student, teacher, indices = rows(5, V, V if K is None else K, torch.float32, "weights", seed=V, listed=K is not None)
    teacher[1, 2], teacher[3, :4] = INF, 3e38
    if indices is not None:
        indices[4, 5], teacher[4, 5] = -1, INF     # (takes no part)
    else:
        student[4, 5], teacher[4, 5] = -INF, INF
    leaf = student.cuda().requires_grad_()
    loss = dsa.topk_distillation(leaf, teacher.cuda(), None if indices is None else indices.cuda(), over=over)
    (d,) = torch.autograd.grad(loss.sum(), leaf)
    cols = torch.arange(V).repeat(5, 1) if indices is None else indices.long()
    assert loss.isnan().tolist() == [False, True, False, True, False]
    for r in range(5):
        assert bool(d[r].cpu()[cols[r]].isnan().all()) == (r in (1, 3)) and (r in (1, 3) or bool(d[r].isfinite().all()))


def test_refusals():
    s, t, i = torch.zeros(4, 10), torch.ones(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    bad = [
        lambda: dsa.topk_distillation(s, t),
        lambda: dsa.topk_distillation(s, t, i.long()),
        lambda: dsa.topk_distillation(s, t, i[:, :2]),
        lambda: dsa.topk_distillation(s, t[:3], i[:3]),
        lambda: dsa.topk_distillation(s.double(), t, i),
        lambda: dsa.topk_distillation(s, t.double(), i),
        lambda: dsa.topk_distillation(s, t, i, teacher_kind="probabilities"),
        lambda: dsa.topk_distillation(s, t, i, over="vocabulary"),
        lambda: dsa.topk_distillation(s, t, i, temperature=0.0),
        lambda: dsa.topk_distillation(s, t, i, temperature=float("inf")),
        lambda: dsa.topk_distillation(s, t, i, temperature=1e-39),
        lambda: dsa.topk_distillation(s, t, i, temperature=float("nan")),
        lambda: dsa.topk_distillation(s[:, ::2], t, i),
        lambda: dsa.topk_distillation(torch.zeros(10, 4).t(), t, i),
        lambda: dsa.topk_distillation(s, torch.ones(3, 4).t(), i),
        lambda: dsa.topk_distillation(s[:, :0], t[:, :0]),
        lambda: dsa.topk_distillation_bwd_raw(s, t, i, torch.zeros(4, 3), torch.zeros(4)),
        lambda: dsa.topk_distillation_bwd_raw(s, t, i, torch.zeros(4, 4), torch.zeros(5)),
    ]
    for call in bad:
        with pytest.raises(ValueError) as e:
            call()
        assert "no CPU path" not in str(e.value), str(e.value)
    with pytest.raises(ValueError, match="no CPU path"):
        dsa.topk_distillation(s, t, i)


def test_c_entry_refuses_before_any_cuda_call():
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    assert lib.dsa_topk_distillation(None, 2, 4, None, 2, None, None, None, 1, 4, 4, 0, 0, 1.0, None, 0, None) != 0
    assert lib.dsa_topk_distillation_bwd(None, 2, 4, None, 2, None, None, None, None, 1, 4, 4, 0, 0, 1.0, None) != 0


def test_c_entry_refuses_a_workspace_off_its_alignment():
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    rows, V, K = 3, 40000, 5
    nbytes = lib.dsa_topk_distillation_workspace_bytes(rows, V, 1, 1)
    assert nbytes > 0
    at = 4096   # (an address that nothing reads: the call is refused before any launch)
    assert lib.dsa_topk_distillation(at, 2, V, at, 2, at, at, at, rows, V, K, 1, 0, 1.0, at + 2, nbytes, None) != 0
    assert b"aligned" in lib.dsa_get_last_error()
