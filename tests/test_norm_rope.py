"""qk_norm_rope / qk_norm_rope_cached against the definition in 64 bits, and what they refuse."""
import itertools

import pytest
import torch

import tilelang_ascend_b200 as dsa

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}   # half a step of the smallest fp16 values


# ------------------------------------------------------------------------------------------------ definition, 64 bits
def rotate(x, positions, inv_freq, start, interleaved, scale, back=False):
    R = 2 * inv_freq.numel()
    angle = positions.double()[:, :, None, None] * inv_freq.double()
    cos, sin = angle.cos() * scale, angle.sin() * scale * (-1 if back else 1)
    part = x[..., start:start + R]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :R // 2], part[..., R // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((x[..., :start], part, x[..., start + R:]), -1)


def norm(x, kind, weight, bias, n, eps):
    if kind is None:
        return x
    h = x[..., :n]
    if kind == "layer":
        h = h - h.mean(-1, keepdim=True)
    h = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        h = h * weight.double()
    if bias is not None:
        h = h + bias.double()
    return torch.cat((h, x[..., n:]), -1)


def reference(x, positions, inv_freq, kind, weight, bias, n, start, interleaved, scale, eps):
    return rotate(norm(x.double(), kind, weight, bias, n, eps), positions, inv_freq, start, interleaved, scale)


def assert_rounded(got, ref, slack, what):
    """got = ref computed in fp32 with an absolute error of at most `slack`, rounded once to its type."""
    got, dt = got.detach().cpu(), got.dtype
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} vs {tuple(ref.shape)}"
    bound = (ref.abs() + slack) * HALF_STEP[dt] + slack + TINY[dt]
    err = (got.double() - ref).abs()
    assert bool((err <= bound).all()), f"{what}: error {float((err - bound).max()):.3g} beyond the bound, largest value {float(ref.abs().max()):.3g}"


# A row's fp32 error: sums of at most 32 sequential and 5 tree additions for the mean square (half of it reaches the reciprocal
# root), one more such sum for a mean, six products and sums after that, cosine and sine within 2^-22: below 64 * 2^-24 of the
# largest |value| that is added up (two members of a pair, each times |cos| + |sin| <= 1.42).
ROW = 64 * 2.0 ** -24


def make(B, S, H, HK, D, R, dtype, seed, far=50000, strided=False):
    g = torch.Generator().manual_seed(seed)
    if strided:
        x = torch.randn((B, S + 1, (H + HK) * D + 16), generator=g).to(dtype)
        q, k = x[:, 1:, :H * D].view(B, S, H, D), x[:, 1:, H * D:(H + HK) * D].view(B, S, HK, D)
    else:
        q, k = (torch.randn((B, S, h, D), generator=g).add(0.3).to(dtype) for h in (H, HK))
    positions = torch.randint(0, far, (B, S), generator=g)
    inv_freq = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float()
    return g, q, k, positions, inv_freq


def on_gpu(t):
    """The same values with the same strides on the GPU."""
    if t is None:
        return None
    out = torch.empty_strided(t.size(), t.stride(), dtype=t.dtype, device="cuda")
    return out.copy_(t)


CASES = [
    # B, S, H, HK, D, R, start, norm_dim, q_norm, k_norm, interleaved
    (1, 1, 1, 1, 128, 64, 0, 128, None, "layer", False),
    (2, 7, 64, 1, 128, 64, 0, 128, None, "layer", True),
    (1, 5, 128, 1, 576, 64, 512, 512, None, "rms", True),
    (1, 5, 128, 1, 576, 64, 512, 512, "rms", "layer", False),
    (3, 11, 6, 2, 192, 192, 0, 192, "rms", "rms", False),
    (1, 300, 3, 3, 64, 32, 32, 40, "layer", "rms", True),       # the norm ends inside the rotated dims
    (2, 9, 5, 1, 1024, 128, 64, 1024, "rms", "rms", False),
    (1, 3, 2, 1, 768, 768, 0, 768, "rms", None, True),
    (1, 130, 4, 4, 256, 16, 8, 256, "rms", "rms", False),
    # no 16-byte units: odd sizes, odd starts
    (2, 5, 3, 2, 90, 30, 7, 61, "rms", "layer", True),
    (1, 4, 2, 1, 101, 100, 1, 101, "layer", "rms", False),
    (1, 3, 1, 1, 2, 2, 0, 1, "rms", None, True),
    (1, 2, 2, 1, 1100, 64, 12, 1100, "layer", "rms", False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case, dtype):
    B, S, H, HK, D, R, start, n, q_norm, k_norm, interleaved = case
    g, q, k, positions, inv_freq = make(B, S, H, HK, D, R, dtype, seed=D + S)
    eps, scale = 1e-5, 1.25
    param_dtype = dtype if D % 3 else torch.float32
    params = {}
    for side, kind in (("q", q_norm), ("k", k_norm)):
        params[side + "_weight"] = (1 + 0.3 * torch.randn(n, generator=g)).to(param_dtype) if kind else None
        params[side + "_bias"] = (0.2 * torch.randn(n, generator=g)).to(param_dtype) if kind == "layer" else None
    leaves = {"q": on_gpu(q).requires_grad_(), "k": on_gpu(k).requires_grad_()}
    leaves.update({name: on_gpu(t).requires_grad_() for name, t in params.items() if t is not None})
    outs = dsa.qk_norm_rope(leaves["q"], leaves["k"], positions.cuda(), inv_freq.cuda(), rope_start=start, interleaved=interleaved, rope_scale=scale,
                            q_norm=q_norm, k_norm=k_norm, norm_dim=n, eps=eps,
                            **{name: leaves.get(name) for name in ("q_weight", "q_bias", "k_weight", "k_bias")})
    d_outs = [torch.randn(o.shape, generator=g).to(dtype) for o in outs]
    torch.autograd.backward(outs, [d.cuda() for d in d_outs])
    for side, x, kind, out, d_out in (("q", q, q_norm, outs[0], d_outs[0]), ("k", k, k_norm, outs[1], d_outs[1])):
        weight, bias = params[side + "_weight"], params[side + "_bias"]
        ref = reference(x, positions, inv_freq, kind, weight, bias, n, start, interleaved, scale, eps)
        assert_rounded(out, ref, ROW * 3 * scale * ref.abs().amax(-1, keepdim=True).clamp(min=1.0), f"{side}'")
        # gradients: autograd through the definition
        d = {"x": x.double().requires_grad_()}
        for name, t in (("weight", weight), ("bias", bias)):
            d[name] = None if t is None else t.double().requires_grad_()
        names = [m for m in ("x", "weight", "bias") if d[m] is not None]
        y = reference(d["x"], positions, inv_freq, kind, d["weight"], d["bias"], n, start, interleaved, scale, eps)
        grads = dict(zip(names, torch.autograd.grad(y, [d[m] for m in names], d_out.double())))
        # |dx| is a sum of three terms, each at most rstd * |weight| * max|u| * max(1, max|n|)
        u = rotate(d_out.double(), positions, inv_freq, start, interleaved, scale, back=True)
        size = u.abs().amax(-1, keepdim=True)
        if kind:
            h = x.double()[..., :n]
            h = h - h.mean(-1, keepdim=True) if kind == "layer" else h
            rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
            unit = h * rstd
            size = size * (1 + rstd * (weight.double().abs().max() * 3 * unit.abs().amax(-1, keepdim=True).clamp(min=1.0)))
        assert_rounded(leaves[side].grad, grads["x"], 2 * ROW * size, f"d{side}")
        if kind:   # sums over all rows: no more sequential additions than rows, plus those of the groups and blocks
            steps = (B * S * x.shape[2] + 64) * 2.0 ** -24 + 2 * ROW
            assert_rounded(leaves[side + "_weight"].grad, grads["weight"], steps * (u[..., :n] * unit).abs().sum((0, 1, 2)) + 1e-12, f"d{side}_weight")
            if bias is not None:
                assert_rounded(leaves[side + "_bias"].grad, grads["bias"], steps * u[..., :n].abs().sum((0, 1, 2)) + 1e-12, f"d{side}_bias")


@pytest.mark.gpu
@pytest.mark.parametrize("D,offset", [(128, 16), (120, 3)])
def test_slices_of_a_projection_are_read_in_place(D, offset):
    """Strided rows, in 16-byte units and not; the gradient of a strided leaf is contiguous."""
    B, S, H, HK = 2, 9, 4, 2
    g = torch.Generator().manual_seed(5)
    fused = torch.randn((B, S, (H + HK) * D + offset), generator=g).to(torch.bfloat16)
    q, k = fused[..., offset:offset + H * D].unflatten(-1, (H, D)), fused[..., offset + H * D:].unflatten(-1, (HK, D))
    dev = fused.cuda()
    qg = dev[..., offset:offset + H * D].unflatten(-1, (H, D)).detach().requires_grad_()
    kg = dev[..., offset + H * D:].unflatten(-1, (HK, D)).detach().requires_grad_()
    positions, inv_freq = torch.arange(S).repeat(B, 1), torch.tensor([1.0, 0.1, 0.01, 1e-3])
    for p in (positions, positions.to(torch.int32)):
        oq, ok = dsa.qk_norm_rope(qg, kg, p.cuda(), inv_freq.cuda(), q_norm="rms", k_norm="rms")
        for got, x in ((oq, q), (ok, k)):
            ref = reference(x, positions, inv_freq, "rms", None, None, D, 0, True, 1.0, 1e-6)
            assert_rounded(got, ref, ROW * 3 * ref.abs().amax(-1, keepdim=True), "rows")
    d = torch.randn(oq.shape, generator=g).to(torch.bfloat16)
    (dq,) = torch.autograd.grad(oq, qg, d.cuda().transpose(1, 2).contiguous().transpose(1, 2))   # a strided upstream gradient
    dense = qg.detach().contiguous().requires_grad_()
    (dq2,) = torch.autograd.grad(dsa.qk_norm_rope(dense, None, positions.cuda(), inv_freq.cuda(), q_norm="rms")[0], dense, d.cuda())
    assert dq.is_contiguous() and torch.equal(dq, dq2)


@pytest.mark.gpu
def test_far_positions_and_gradient_by_differences():
    """Angles of positions past 32 bits, and the gradient against central differences of the 64-bit definition."""
    g, q, _, _, inv_freq = make(1, 6, 2, 1, 64, 64, torch.float16, seed=3)
    positions = torch.tensor([[0, 1, -7, 1_000_003, (1 << 31) + 5, (1 << 40) + 12345]])
    leaf = q.cuda().requires_grad_()
    out, none = dsa.qk_norm_rope(leaf, None, positions.cuda(), inv_freq.cuda(), q_norm="rms", interleaved=False)
    assert none is None
    ref = reference(q, positions, inv_freq, "rms", None, None, 64, 0, False, 1.0, 1e-6)
    # an angle of 2^40 carries 2^-12 of its 52 bits' step into the reference's own reduction: 2^-13 radians are not held apart there
    slack = ROW * 3 * ref.abs().amax(-1, keepdim=True) + torch.tensor([0, 0, 0, 0, 2.0 ** -21, 2.0 ** -12]).view(1, 6, 1, 1) * 3
    assert_rounded(out, ref, slack, "far")
    d = torch.randn(out.shape, generator=g, dtype=torch.float64)
    (grad,) = torch.autograd.grad(out, leaf, d.to(torch.float16).cuda())
    h = 1e-5
    for at in ((0, 0, 0, 0), (0, 2, 1, 37), (0, 3, 0, 63)):
        step = torch.zeros(q.shape, dtype=torch.float64)
        step[at] = h
        hi, lo = (norm_rope_64(q.double() + s, positions, inv_freq) for s in (step, -step))
        want = float(((hi - lo) * d.to(torch.float16).double()).sum() / (2 * h))
        assert abs(float(grad[at]) - want) <= abs(want) * 2.0 ** -11 + 1e-4


def norm_rope_64(x, positions, inv_freq):
    return rotate(norm(x, "rms", None, None, x.shape[-1], 1e-6), positions, inv_freq, 0, False, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("parts,D,start,slot_dtype", [(2, 576, 512, torch.int32), (1, 576, 512, torch.int64), (1, 128, 0, torch.int32), (2, 90, 60, torch.int32)])
def test_cached_rows_go_to_their_slots_and_no_others(parts, D, start, slot_dtype):
    B, S, H, HK, R = 3, 5, 4, 2, (30 if D == 90 else 64)
    g, q, k, positions, inv_freq = make(B, S, H, HK, D, R, torch.bfloat16, seed=D)
    n = start if start else D
    weight = 1 + 0.1 * torch.randn(n, generator=g)
    blocks, bs = 4, 16
    slots = torch.randperm(blocks * bs, generator=g)[:B * S].view(B, S).to(slot_dtype)
    slots[0, 3], slots[2, 0], slots[1, 1] = -1, blocks * bs, torch.iinfo(slot_dtype).min
    split = D - R if parts == 2 else D
    cache, tail = torch.randn((blocks, bs, HK, split), generator=g).to(torch.bfloat16), torch.randn((blocks, bs, HK, R), generator=g).to(torch.bfloat16)
    cg, tg = cache.cuda(), tail.cuda()
    kw = dict(rope_start=start, k_norm="rms", k_weight=weight.cuda(), norm_dim=n)
    out = dsa.qk_norm_rope_cached(q.cuda(), k.cuda(), positions.cuda(), inv_freq.cuda(), cg, slots.cuda(), key_cache_rope=tg if parts == 2 else None, **kw)
    oq, ok = dsa.qk_norm_rope(q.cuda(), k.cuda(), positions.cuda(), inv_freq.cuda(), **kw)
    assert torch.equal(out, oq)
    want, want_tail = cache.clone().view(-1, HK, split), tail.clone().view(-1, HK, R)
    for b, s in itertools.product(range(B), range(S)):
        slot = int(slots[b, s])
        if 0 <= slot < blocks * bs:
            want[slot] = ok[b, s, :, :split].cpu()
            if parts == 2:
                want_tail[slot] = ok[b, s, :, split:].cpu()
    assert torch.equal(cg.cpu().view_as(want), want) and torch.equal(tg.cpu().view_as(want_tail), want_tail)
    # keys alone
    cg2 = cache.cuda()
    assert dsa.qk_norm_rope_cached(None, k.cuda(), positions.cuda(), inv_freq.cuda(), cg2, slots.cuda(), key_cache_rope=tg if parts == 2 else None, **kw) is None
    assert torch.equal(cg2, cg)


@pytest.mark.gpu
def test_a_bias_without_a_weight_and_rows_used_twice():
    g, q, _, positions, inv_freq = make(2, 4, 3, 1, 128, 64, torch.bfloat16, seed=21)
    bias = (0.3 * torch.randn(128, generator=g)).float()
    leaf, b = q.cuda().requires_grad_(), bias.cuda().requires_grad_()
    oq, ok = dsa.qk_norm_rope(leaf, leaf, positions.cuda(), inv_freq.cuda(), q_norm="layer", q_bias=b)
    (oq.float().sum() * 2 + ok.float().sum()).backward()
    x, bd = q.double().requires_grad_(), bias.double().requires_grad_()
    ref = reference(x, positions, inv_freq, "layer", None, bd, 128, 0, True, 1.0, 1e-6)
    assert_rounded(oq, ref.detach(), ROW * 3 * ref.detach().abs().amax(-1, keepdim=True), "q'")
    two = reference(x, positions, inv_freq, None, None, None, 128, 0, True, 1.0, 1e-6)
    dx, db = torch.autograd.grad(ref.sum() * 2 + two.sum(), (x, bd))
    # two gradients of the leaf, each rounded, and their sum: 3 half steps of the two parts (each at most 3, the norm's terms cancel)
    assert float((leaf.grad.cpu().double() - dx).abs().max()) <= 3 * 2.0 ** -8 * 6
    assert_rounded(b.grad, db, 1e-4, "dbias")
    # a side whose output is not used asks for nothing
    leaf2, k2 = q.cuda().requires_grad_(), q.cuda().requires_grad_()
    oq, ok = dsa.qk_norm_rope(leaf2, k2, positions.cuda(), inv_freq.cuda(), q_norm="rms", k_norm="rms")
    ok.sum().backward()
    assert leaf2.grad is None and k2.grad is not None


@pytest.mark.gpu
def test_masked_values_and_empty_calls():
    """Infinities and NaN stay in their own row; calls without tokens return empty tensors; the sums of no rows are zeros."""
    _, q, k, positions, inv_freq = make(1, 6, 3, 1, 128, 64, torch.bfloat16, seed=8)
    clean = dsa.qk_norm_rope(q.cuda(), k.cuda(), positions.cuda(), inv_freq.cuda(), q_norm="rms", k_norm="layer")[0]
    bad = q.clone()
    bad[0, 2, 1, 5], bad[0, 4, 0, 100] = float("inf"), float("nan")
    got = dsa.qk_norm_rope(bad.cuda(), k.cuda(), positions.cuda(), inv_freq.cuda(), q_norm="rms", k_norm="layer")[0]
    same = torch.ones(1, 6, 3, dtype=torch.bool)
    same[0, 2, 1] = same[0, 4, 0] = False
    assert torch.equal(got.cpu()[same], clean.cpu()[same]) and bool(got.cpu()[~same].isnan().any(-1).all())
    zero = dsa.qk_norm_rope(torch.zeros_like(q).cuda(), None, positions.cuda(), inv_freq.cuda(), q_norm="rms")[0]
    assert bool((zero == 0).all())
    empty = torch.empty((0, 6, 3, 128), dtype=torch.bfloat16, device="cuda", requires_grad=True)
    weight = torch.ones(128, device="cuda", requires_grad=True)
    out, _ = dsa.qk_norm_rope(empty, None, positions[:0].cuda(), inv_freq.cuda(), q_norm="rms", q_weight=weight)
    assert out.shape == empty.shape
    out.sum().backward()
    assert bool((weight.grad == 0).all())


@pytest.mark.gpu
def test_repeatable_captured_and_on_another_stream():
    _, q, k, positions, inv_freq = make(2, 50, 8, 2, 128, 128, torch.bfloat16, seed=9)
    q, k, positions, inv_freq = q.cuda(), k.cuda(), positions.cuda(), inv_freq.cuda()
    weight = torch.linspace(0.5, 1.5, 128, device="cuda")
    d = torch.randn(q.shape, device="cuda").to(q.dtype)

    def step():
        oq, ok = dsa.qk_norm_rope(q, k, positions, inv_freq, q_norm="rms", k_norm="rms", q_weight=weight, interleaved=False)
        grads = dsa.qk_norm_rope_bwd_raw(d, k * 0.5, q, None, positions, inv_freq, q_norm="rms", q_weight=weight, interleaved=False)
        return (oq, ok) + grads[:3]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


@pytest.mark.gpu
def test_gradient_of_one_side_alone():
    """A side without a gradient is left out, whatever else is given for it."""
    g = torch.Generator().manual_seed(5)
    q, k, d_q, d_k = (torch.randn((2, 9, h, 64), generator=g).to(torch.bfloat16).cuda() for h in (4, 1, 4, 1))
    pos, f = torch.arange(18, dtype=torch.int32).view(2, 9).cuda(), torch.rand(16, generator=g).cuda()
    w = torch.rand(64, generator=g).cuda()
    how = dict(q_norm="rms", k_norm="layer", q_weight=w, k_weight=w, k_bias=w)
    both = dsa.qk_norm_rope_bwd_raw(d_q, d_k, q, k, pos, f, **how)
    keys, queries = dsa.qk_norm_rope_bwd_raw(None, d_k, q, k, pos, f, **how), dsa.qk_norm_rope_bwd_raw(d_q, None, q, k, pos, f, **how)
    assert all(keys[i] is None for i in (0, 2, 3)) and all(torch.equal(keys[i], both[i]) for i in (1, 4, 5))
    assert all(queries[i] is None for i in (1, 3, 4, 5)) and all(torch.equal(queries[i], both[i]) for i in (0, 2))


def check_one_side(kind, B, S, H, D, R, start, n, interleaved, dtype, eps, seed):
    """Output and gradients of queries alone against autograd through the definition (on the GPU, in 64 bits); upstream gradients above 0, so that rows
    missing from the parameters' sums would show."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, S, H, D), generator=g).add(0.3).to(dtype).cuda()
    d_out = torch.rand((B, S, H, D), generator=g).add(0.5).to(dtype).cuda()
    weight, bias = (1 + 0.3 * torch.randn(n, generator=g)).cuda(), (0.2 * torch.randn(n, generator=g)).cuda() if kind == "layer" else None
    positions = torch.randint(0, 50000, (B, S), generator=g).cuda()
    inv_freq = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().cuda()
    names, leaves = (("x", "weight", "bias"), (x, weight, bias)) if bias is not None else (("x", "weight"), (x, weight))
    mine = [t.detach().requires_grad_() for t in leaves]
    out, _ = dsa.qk_norm_rope(mine[0], None, positions, inv_freq, rope_start=start, interleaved=interleaved, q_norm=kind, q_weight=mine[1],
                              q_bias=mine[2] if bias is not None else None, norm_dim=n, eps=eps)
    got = dict(zip(names, torch.autograd.grad(out, mine, d_out)))
    exact = [t.double().requires_grad_() for t in leaves]
    y = reference(exact[0], positions, inv_freq, kind, exact[1], exact[2] if bias is not None else None, n, start, interleaved, 1.0, eps)
    want = dict(zip(names, torch.autograd.grad(y, exact, d_out.double())))
    y = y.detach()
    assert_rounded(out, y.cpu(), (ROW * 3 * y.abs().amax(-1, keepdim=True).clamp(min=1.0)).cpu(), "rows")
    h = x.double()[..., :n]
    h = h - h.mean(-1, keepdim=True) if kind == "layer" else h
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = h * rstd
    most = unit.abs().amax(-1, keepdim=True).clamp(min=1.0)
    u = rotate(d_out.double(), positions, inv_freq, start, interleaved, 1.0, back=True)
    size = u.abs().amax(-1, keepdim=True) * (1 + rstd * (weight.double().abs().max() * 3 * most))
    assert_rounded(got["x"], want["x"].cpu(), (2 * ROW * size).cpu(), "dx")
    # sums over the rows: those of a block in turn at most (296 blocks), its groups, the blocks' lines.  A term u n is off by |u| times 2 ROW of the
    # row's largest |n|, and by |n| times what u is off by: u = a cos + b sin with |a| + |b| <= 2 max|u| (a rotation of a pair of u), cosine and sine
    # within 4 * 2^-24, two roundings: 12 * 2^-24 max|u| < ROW max|u|, however small u itself is
    additions = (B * S * H / 296 + 128) * 2.0 ** -24
    umax, u = ROW * u.abs().amax(-1, keepdim=True), u[..., :n].abs()
    terms = additions * u * unit.abs() + 2 * ROW * u * most + umax * unit.abs()
    assert_rounded(got["weight"], want["weight"].cpu(), terms.sum((0, 1, 2)).cpu(), "dweight")
    if bias is not None:
        assert_rounded(got["bias"], want["bias"].cpu(), (additions * u + umax).sum((0, 1, 2)).cpu(), "dbias")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("B,S,H,D,R,start,n,interleaved", [
    (1, 1, 1, 128, 64, 0, 128, False),     # one row
    (2, 7, 3, 64, 64, 0, 64, True),        # rows that do not fill a block's groups
    (1, 5, 1, 576, 64, 512, 512, True),
    (1, 300, 3, 256, 64, 192, 192, False),
    (1, 3, 2, 90, 30, 7, 61, True),        # element by element
])
def test_gradients_without_eps(B, S, H, D, R, start, n, interleaved, kind, dtype):
    check_one_side(kind, B, S, H, D, R, start, n, interleaved, dtype, 0.0, seed=D + S)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,B,S,H,D,R,start,n,interleaved", [
    ("rms", 2, 1201, 16, 128, 128, 0, 128, False),
    ("layer", 1, 10007, 1, 576, 64, 512, 512, True),
    ("layer", 3, 2003, 13, 64, 64, 0, 64, True),
    ("rms", 1, 5003, 2, 90, 30, 7, 61, False),       # element by element
])
def test_parameter_gradients_over_more_rows_than_fit_the_chip(kind, B, S, H, D, R, start, n, interleaved):
    """More tiles of rows than blocks: a block's sums go over several of them."""
    check_one_side(kind, B, S, H, D, R, start, n, interleaved, torch.bfloat16, 1e-6, seed=D)


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_slots_and_of_a_side_alone():
    q, k = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    pos, f, w = torch.zeros(2, 3, dtype=torch.int32), torch.ones(16), torch.ones(64)
    with pytest.raises(ValueError, match="slots"):
        dsa.qk_norm_rope_cached(q, k, pos, f, torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16), [[0, 1, 2], [3, 4, 5]])
    with pytest.raises(ValueError, match="no CPU path"):   # (everything else is in order)
        dsa.qk_norm_rope_bwd_raw(None, k, q, k, pos, f, q_norm="rms", q_weight=w, k_norm="rms", k_weight=w)


def test_refusals():
    q, k = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    pos, f = torch.zeros(2, 3, dtype=torch.int32), torch.ones(16)
    cache, slots = torch.zeros(2, 8, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32)
    w = torch.ones(64)
    bad = [
        lambda: dsa.qk_norm_rope(None, None, pos, f),
        lambda: dsa.qk_norm_rope(q[0], None, pos, f),
        lambda: dsa.qk_norm_rope(q, k[:, :2], pos, f),
        lambda: dsa.qk_norm_rope(q, k.half(), pos, f),
        lambda: dsa.qk_norm_rope(q.float(), None, pos, f),
        lambda: dsa.qk_norm_rope(q.transpose(2, 3), None, pos, f),
        lambda: dsa.qk_norm_rope(q, k, pos.float(), f),
        lambda: dsa.qk_norm_rope(q, k, pos[0], f),
        lambda: dsa.qk_norm_rope(q, k, pos, f.double()),
        lambda: dsa.qk_norm_rope(q, k, pos, torch.ones(33)),
        lambda: dsa.qk_norm_rope(q, k, pos, torch.ones(0)),
        lambda: dsa.qk_norm_rope(q, k, pos, f, rope_start=34),
        lambda: dsa.qk_norm_rope(q, k, pos, f, rope_start=-2),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_norm="rms", norm_dim=0),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_norm="batch"),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_weight=w),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_norm="rms", q_weight=w[:32]),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_norm="rms", q_weight=w.double()),
        lambda: dsa.qk_norm_rope(q, k, pos, f, q_norm="layer", q_weight=w, q_bias=w.bfloat16()),
        lambda: dsa.qk_norm_rope_cached(q, None, pos, f, cache, slots),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache, slots.float()),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache, slots[:1]),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache[..., :32].contiguous(), slots),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache[..., :32].contiguous(), slots, key_cache_rope=cache[..., :32].contiguous(), rope_start=0),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache.half(), slots),
        lambda: dsa.qk_norm_rope_cached(q, k, pos, f, cache[:, ::2], slots),
        lambda: dsa.qk_norm_rope_cached(q.requires_grad_(), k, pos, f, cache, slots),
        lambda: dsa.qk_norm_rope_bwd_raw(k, None, q.detach(), None, pos, f, q_norm="rms"),
        lambda: dsa.qk_norm_rope_bwd_raw(k, None, None, None, pos, f, q_norm="rms"),
        lambda: dsa.qk_norm_rope_bwd_raw(None, None, q.detach(), k, pos, f),
    ]
    for call in bad:
        with pytest.raises(ValueError) as e:
            call()
        assert "no CPU path" not in str(e.value), str(e.value)
    with pytest.raises(ValueError, match="no CPU path"):
        dsa.qk_norm_rope(q.detach(), k, pos, f)


def test_c_entry_refuses_before_any_cuda_call():
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    scalars = (None, 0, None, 1, 1, 64, 32, 0, 0, 1, 1.0, 1e-6)
    assert lib.dsa_norm_rope(None, None, *scalars, 0, None) != 0 and b"given" in lib.dsa_get_last_error()
    assert lib.dsa_norm_rope_bwd(None, None, *scalars, None, 0, 0, None) != 0


def test_c_entry_refuses_a_workspace_off_its_alignment():
    from ctypes import byref
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    at = 4096   # (an address that nothing reads: the call is refused before any launch)
    rows = _lib.RopeRows(at, 64, 64, 64, 1, 1, at, None, 1, 64, at, None, None, 0, 0, 0)
    side = _lib.RopeGrads(rows, at, 64, 64, 64, at, None)
    assert lib.dsa_norm_rope_bwd(byref(side), None, at, 0, at, 1, 1, 64, 32, 0, 64, 1, 1.0, 1e-6, at + 1, 1 << 30, 0, None) != 0
    assert b"aligned" in lib.dsa_get_last_error()
