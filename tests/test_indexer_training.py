"""What trains the lightning indexer: the teacher's weights of the listed keys, the gradient of the listed scores, and both in a
training step with the rest of the path -- against the definitions in 64 bits."""
import pytest
import torch

import tilelang_ascend_b200 as dsa

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
INF = float("inf")


def check_status():
    assert dsa.kernel_status() == 0, "a bounded in-kernel wait gave up"


def lists(g, B, S, S_kv, K, holes=True):
    """Causal lists of distinct keys, shorter than K where a query has fewer keys; with holes, keys that do not exist and, in the
    last sequence, a query without keys."""
    out = torch.full((B, S, 1, K), -1, dtype=torch.int32)
    for b in range(B):
        for s in range(S):
            n = max(S_kv - S + 1 + s, 0)
            keys = torch.randperm(n, generator=g)[:K].to(torch.int32)
            out[b, s, 0, torch.randperm(K, generator=g)[:keys.numel()]] = keys
    if holes and K > 2:
        out[0, 0, 0, 1] = S_kv
        out[0, 0, 0, K - 1] = -5
        if S > 1:
            out[-1, 1] = -1
    return out


# ------------------------------------------------------------------------------------------------- weights of the keys
def key_weights(q, kv, indices, lse, scale, q_start):
    """The definition, and a bound of its fp32 error."""
    B, S, H, D = q.shape
    out, slack = torch.zeros(indices.shape, dtype=torch.float64), torch.zeros(indices.shape, dtype=torch.float64)
    for b in range(B):
        for s in range(S):
            idx = indices[b, s, 0].long()
            there = (idx >= 0) & (idx < kv.shape[1]) & (idx <= q_start + s)
            rows, heads = kv[b, idx[there], 0].double(), q[b, s].double()
            l = lse[b, s].double()
            w = torch.exp(rows @ heads.T * scale - torch.where(l == -INF, INF, l))
            out[b, s, 0, there] = w.mean(1)
            # the exponent: a sum of D products in steps of 16, each within 2^-22 of what has been summed up; the normaliser and its
            # difference 3 steps; the exponential itself 2^-22; H additions
            size = rows.abs() @ heads.abs().T * scale * (D / 16 + 1) * 2.0 ** -22 + (l.abs().nan_to_num(posinf=0) + 8) * 3 * 2.0 ** -24 + 2.0 ** -21
            slack[b, s, 0, there] = (w * size).mean(1) + w.mean(1) * H * 2.0 ** -24
    return out, slack


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,S_kv,H,D,K", [
    (1, 1, 1, 1, 576, 1),            # one key, one head
    (1, 3, 200, 128, 576, 128),
    (2, 5, 70, 16, 576, 129),        # more slots than keys; a last tile of one entry
    (1, 4, 900, 64, 576, 700),
    (2, 3, 300, 40, 512, 257),       # heads that are not a multiple of 16, no rotated part
    (1, 2, 260, 200, 576, 256),      # two passes over the heads
    (1, 2, 300, 24, 640, 260),       # widest rows
    (1, 3, 150, 6, 72, 100),         # rows that end inside a chunk
    (1, 2, 9000, 128, 576, 8192),    # longest lists
])
def test_key_weights(B, S, S_kv, H, D, K, dtype):
    g = torch.Generator().manual_seed(S_kv + K)
    q, kv = torch.randn((B, S, H, D), generator=g).to(dtype), torch.randn((B, S_kv, 1, D), generator=g).to(dtype)
    indices = lists(g, B, S, S_kv, K)
    lse = torch.randn((B, S, H), generator=g) + 5
    if H > 2:
        lse[0, 0, 1] = -INF          # a head that saw no key
    scale = 0.9 * D ** -0.5
    got = dsa.sparse_mla_key_weights(q.cuda(), kv.cuda(), indices.cuda(), lse.cuda(), sm_scale=scale)
    check_status()
    want, slack = key_weights(q, kv, indices, lse, scale, S_kv - S)
    assert got.shape == (B, S, 1, K) and got.dtype == torch.float32 and not got.requires_grad
    err = (got.cpu().double() - want).abs()
    assert bool((err <= slack).all()), f"off by {float((err - slack).max()):.3g}, largest weight {float(want.max()):.3g}"
    assert not got.cpu()[want == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S,S_kv,H,D,K", [
    (1, 460, 700, 64, 576, 300),     # three to four queries in turn on every SM
    (2, 301, 500, 128, 576, 257),
    (1, 450, 600, 200, 576, 384),    # two passes over the heads
    (1, 450, 500, 128, 640, 200),    # widest rows: three stages
    (1, 1000, 1000, 24, 512, 130),   # causal from the first key on: lists of one tile and of two
])
def test_key_weights_of_more_queries_than_sms(B, S, S_kv, H, D, K, dtype):
    """Queries that follow one another on an SM, queries without keys between them: against the definition on the GPU in 64 bits."""
    g = torch.Generator().manual_seed(S + H)
    q, kv = torch.randn((B, S, H, D), generator=g).to(dtype).cuda(), torch.randn((B, S_kv, 1, D), generator=g).to(dtype).cuda()
    indices = lists(g, B, S, S_kv, K)
    gone = torch.rand((B, S), generator=g) < 0.2
    gone[:, S // 2:S // 2 + 3] = True
    indices[gone] = -1
    indices[-1, S - 9, 0, 128:] = -1          # a list that ends with its first tile
    indices[-1, S - 8, 0, :128] = -1          # one that begins with its second
    indices = indices.cuda()
    lse = (torch.randn((B, S, H), generator=g) + 5).cuda()
    lse[0, ::7, 1] = -INF
    scale = 0.9 * D ** -0.5
    got = dsa.sparse_mla_key_weights(q, kv, indices, lse, sm_scale=scale)
    again = dsa.sparse_mla_key_weights(q, kv, indices, lse, sm_scale=scale)
    check_status()
    assert torch.equal(got, again)
    last = torch.arange(S, device="cuda") + (S_kv - S)
    for b in range(B):
        for s0 in range(0, S, 50):
            idx = indices[b, s0:s0 + 50, 0].long()
            there = (idx >= 0) & (idx < S_kv) & (idx <= last[s0:s0 + 50, None])
            rows, heads = kv[b, idx.clamp(0, S_kv - 1), 0].double(), q[b, s0:s0 + 50].double()
            l = lse[b, s0:s0 + 50].double()[:, :, None]
            w = torch.exp(heads @ rows.transpose(1, 2) * scale - torch.where(l == -INF, INF, l))
            # (the bound of key_weights)
            size = heads.abs() @ rows.abs().transpose(1, 2) * scale * (D / 16 + 1) * 2.0 ** -22 + (l.abs().nan_to_num(posinf=0) + 8) * 3 * 2.0 ** -24 + 2.0 ** -21
            want = torch.where(there, w.mean(1), 0.0)
            slack = torch.where(there, (w * size).mean(1) + w.mean(1) * H * 2.0 ** -24, 0.0)
            err = (got[b, s0:s0 + 50, 0].double() - want).abs()
            assert bool((err <= slack).all()), f"sequence {b}, queries from {s0}: off by {float((err - slack).max()):.3g}, largest weight {float(want.max()):.3g}"


@pytest.mark.gpu
def test_key_weights_are_the_forwards_softmax():
    """With the forward's own normalisers a list's weights add up to 1, and those of one head give its output."""
    g = torch.Generator().manual_seed(2)
    B, S, S_kv, K = 1, 6, 500, 256
    for H in (1, 128):
        q, kv = torch.randn((B, S, H, 576), generator=g).to(torch.bfloat16).cuda(), torch.randn((B, S_kv, 1, 576), generator=g).to(torch.bfloat16).cuda()
        indices = lists(g, B, S, S_kv, K, holes=False).cuda()
        out, lse = dsa.sparse_mla(q, kv, indices)
        w = dsa.sparse_mla_key_weights(q, kv, indices, lse)
        check_status()
        # H exponentials and the normaliser, each within a few 2^-22 of theirs
        assert float((w.sum(-1) - 1).abs().max()) < 2.0 ** -16
        if H == 1:
            rows = kv[0, indices[0, :, 0].long().clamp(min=0), 0, :512].double()
            by_hand = torch.einsum("sk,skd->sd", w[0, :, 0].double(), rows)
            # the forward rounds its weights and its output to bf16
            assert float((out[0, :, 0].double() - by_hand).abs().max()) < 2.0 ** -7 * float(rows.abs().max())


@pytest.mark.gpu
def test_key_weights_mask_values_in_places_that_take_no_part():
    g = torch.Generator().manual_seed(4)
    q, kv = torch.randn((1, 4, 16, 576), generator=g).to(torch.bfloat16), torch.randn((1, 64, 1, 576), generator=g).to(torch.bfloat16)
    indices = lists(g, 1, 4, 64, 40)
    indices[0, :, 0][indices[0, :, 0] == 7] = -1
    lse = torch.randn((1, 4, 16), generator=g) + 4
    clean = dsa.sparse_mla_key_weights(q.cuda(), kv.cuda(), indices.cuda(), lse.cuda())
    kv[0, 7], kv[0, 63, 0, 3] = float("nan"), INF      # key 7 is listed by nobody, key 63 lies behind all but the last query
    indices[0, :3, 0, 5] = 63
    got = dsa.sparse_mla_key_weights(q.cuda(), kv.cuda(), indices.cuda(), lse.cuda())
    check_status()
    keep = torch.ones(40, dtype=torch.bool)
    keep[5] = False
    assert torch.equal(got[0, :3, 0][:, keep.cuda()], clean[0, :3, 0][:, keep.cuda()]) and not got[0, :3, 0, 5].any()
    assert not dsa.sparse_mla_key_weights(q.cuda(), kv.cuda(), torch.full_like(indices, -1).cuda(), lse.cuda()).any()
    empty = dsa.sparse_mla_key_weights(q[:, :0].cuda(), kv.cuda(), indices[:, :0].cuda(), lse[:, :0].cuda())
    assert empty.shape == (1, 0, 1, 40)


# ------------------------------------------------------------------------------------------ gradient of listed scores
def indexer_gradients(query, key, weights, indices, d_values):
    """The definition: gradients in 64 bits, and bounds of what rounding dz to the inputs' type and summing in fp32 make of them."""
    B, S1, N1, _ = query.shape
    half = HALF_STEP[query.dtype]
    out = {n: torch.zeros(t.shape, dtype=torch.float64) for n, t in (("q", query), ("k", key), ("w", weights))}
    err = {n: torch.zeros_like(t) for n, t in out.items()}
    for b in range(B):
        for s in range(S1):
            idx = indices[b, s, 0].long()
            there = (idx >= 0) & (idx < key.shape[1])
            idx, g = idx[there], d_values[b, s, 0][there].double()
            rows, heads, w = key[b, idx, 0].double(), query[b, s].double(), weights[b, s].double()
            z = rows @ heads.T
            out["w"][b, s] = g @ z.clamp(min=0)
            err["w"][b, s] = (g.abs() @ z.clamp(min=0)) * (idx.numel() / 128 + 16) * 2.0 ** -23
            dz = torch.where(z > 0, g[:, None] * w, torch.zeros_like(z))
            # one rounding of each dz (fp16: also half a step of its smallest values, relative to the list's largest); a z whose sign fp32
            # cannot tell may go either way
            near = (z.abs() <= rows.abs() @ heads.abs().T * 9 * 2.0 ** -22) & (z != 0)
            top = float(g.abs().max() * w.abs().max()) if g.numel() else 0.0
            off = dz.abs() * half + near * (g[:, None] * w).abs() + (2.0 ** -24 * top if query.dtype == torch.float16 else 0.0)
            err["w"][b, s] += (g.abs()[:, None] * near * z.abs()).sum(0)
            sums = (idx.numel() / 16 + 8) * 2.0 ** -22
            out["q"][b, s] = dz.T @ rows
            err["q"][b, s] = off.T @ rows.abs() + sums * (dz.abs().T @ rows.abs())
            out["k"][b, :, 0].index_add_(0, idx, dz @ heads)
            err["k"][b, :, 0].index_add_(0, idx, off @ heads.abs() + (S1 + 8) * 2.0 ** -22 * (dz.abs() @ heads.abs()))
    return out, err


def eight_bit(x):
    """Multiples of 1/16 up to 8: products and their sums are exact in fp32, so is the sign of every z."""
    return (x * 16).round().clamp(-128, 127) / 16


def make_indexer(g, B, S1, S2, N1, K, dtype, exact_signs=True):
    query, key = torch.randn((B, S1, N1, 128), generator=g), torch.randn((B, S2, 1, 128), generator=g)
    if exact_signs:
        query, key = eight_bit(query), eight_bit(key)
    weights = torch.randn((B, S1, N1), generator=g) / (8 * N1)
    return query.to(dtype), key.to(dtype), weights, lists(g, B, S1, S2, K)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S1,S2,N1,K,exact_signs", [
    (1, 1, 1, 1, 1, True),
    (1, 3, 40, 64, 128, True),       # more slots than keys
    (2, 5, 300, 32, 129, True),      # a last tile of one entry
    (1, 2, 700, 16, 512, False),
    (2, 7, 64, 8, 200, True),
    (1, 5, 3000, 64, 2048, True),
    (1, 2, 9000, 40, 8192, True),    # longest lists, heads that are not a power of two
    (3, 40, 250, 64, 100, False),
])
def test_gradient_of_listed_scores(B, S1, S2, N1, K, exact_signs, dtype):
    g = torch.Generator().manual_seed(S2 + N1)
    query, key, weights, indices = make_indexer(g, B, S1, S2, N1, K, dtype, exact_signs)
    d_values = torch.randn(indices.shape, generator=g) * 1e-3 * 10.0 ** torch.randint(-4, 3, (B, S1, 1, 1), generator=g)
    d_values[(indices < 0) | (indices >= S2)] = float("nan")
    dq, dk, dw = dsa.lightning_indexer_bwd_raw(query.cuda(), key.cuda(), weights.cuda(), indices.cuda(), d_values.cuda())
    check_status()
    want, err = indexer_gradients(query, key, weights, indices, d_values)
    half = HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, got, bound in (("q", dq, err["q"] + (want["q"].abs() + err["q"]) * half + tiny), ("k", dk, err["k"]), ("w", dw, err["w"])):
        off = (got.cpu().double() - want[name]).abs()
        assert got.shape == want[name].shape and bool((off <= bound + 1e-30).all()), f"d{name} off by {float((off - bound).max()):.3g}, largest {float(want[name].abs().max()):.3g}"
    assert dq.dtype == dtype and dk.dtype == torch.float32 and dw.dtype == torch.float32


def relative(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("B,S1,S2,N1,K", [(1, 2050, 700, 64, 600), (2, 1030, 1290, 32, 700), (3, 1400, 1061, 16, 1061), (1, 1600, 1600, 64, 1300)])
def test_gradient_of_lists_that_hold_most_keys(B, S1, S2, N1, K):
    """Long lists of many queries, whose gradients are summed tile by tile: against the definition on the GPU in 64 bits, with holes, keys listed twice,
    queries without keys and padding that was never written."""
    from tilelang_ascend_b200 import _lib
    assert _lib.load().dsa_lightning_indexer_bwd_workspace_bytes(B, S1, S2, N1, 128, K, _lib.DTYPE_BF16) > 0   # (that way, then)
    g = torch.Generator().manual_seed(S1 + N1)
    query, key, weights, _ = make_indexer(g, B, S1, S2, N1, 4, torch.bfloat16)
    if S1 <= S2:
        indices = lists(g, B, S1, S2, K)
    else:
        indices = torch.stack([torch.randperm(S2, generator=g)[:K] for _ in range(B * S1)]).view(B, S1, 1, K).to(torch.int32)
    indices[0, 3, 0, 5:40] = indices[0, 3, 0, 45:80]
    indices[0, 7:20] = -1
    query, key, weights, indices = (t.cuda() for t in (query, key, weights, indices))
    d_values = torch.randn(indices.shape, generator=g).cuda() * 1e-3
    there = (indices >= 0) & (indices < S2)
    d_values[~there] = float("nan")
    # the definition: a dense matrix of gradients (entries of one key add up)
    dense = torch.zeros((B, S1, S2), dtype=torch.float64, device="cuda")
    dense.view(B * S1, S2).scatter_add_(1, indices.view(B * S1, K).clamp(0, S2 - 1).long(), torch.where(there, d_values, torch.zeros_like(d_values)).double().view(B * S1, K))
    want = [torch.zeros(t.shape, dtype=torch.float64) for t in (query, key, weights)]
    for b in range(B):
        for s in range(0, S1, 50):
            q, gr, w = query[b, s:s + 50].double(), dense[b, s:s + 50], weights[b, s:s + 50].double()
            z = torch.einsum("shd,kd->shk", q, key[b, :, 0].double())
            want[2][b, s:s + 50] = (z.clamp(min=0) * gr[:, None]).sum(2).cpu()
            dz = (z > 0) * gr[:, None] * w[:, :, None]
            want[0][b, s:s + 50] = torch.einsum("shk,kd->shd", dz, key[b, :, 0].double()).cpu()
            want[1][b, :, 0] += torch.einsum("shk,shd->kd", dz, q).cpu()
    # norms: dz rounded once (2^-8 at most, of every term), dq once more; dw in fp32
    bounds = (2 * 2.0 ** -8, 2.0 ** -8, 2.0 ** -18)
    for name, got, ref, bound in zip("qkw", dsa.lightning_indexer_bwd_raw(query, key, weights, indices, d_values), want, bounds):
        assert relative(got, ref) <= bound, f"d{name} off by {relative(got, ref):.3g} of its norm"
        assert name != "q" or not got[0, 7:20].any()
    check_status()
    # keys that nobody lists and queries without a list may hold anything
    taken = torch.zeros((B, S2), dtype=torch.bool, device="cuda")
    taken.scatter_(1, torch.where(there, indices, torch.zeros_like(indices)).view(B, -1).long(), True)
    dirty_key, dirty_query = key.clone(), query.clone()
    if not bool(taken.all()):
        dirty_key[~taken] = float("nan")
    dirty_query[0, 9] = INF
    for name, got, ref, bound in zip("qkw", dsa.lightning_indexer_bwd_raw(dirty_query, dirty_key, weights, indices, d_values), want, bounds):
        assert relative(got, ref) <= bound, f"d{name} with unwritten padding off by {relative(got, ref):.3g} of its norm"
    check_status()


@pytest.mark.gpu
def test_gradient_of_very_many_queries():
    """More than 2^16 blocks of 128 (query, head) rows, whose places no 16-bit number holds."""
    g = torch.Generator(device="cuda").manual_seed(31)
    S1, S2, N1 = 135001, 96, 64
    query = torch.randn((1, S1, N1, 128), generator=g, device="cuda", dtype=torch.bfloat16)
    key = torch.randn((1, S2, 1, 128), generator=g, device="cuda", dtype=torch.bfloat16)
    weights = torch.randn((1, S1, N1), generator=g, device="cuda")
    indices = torch.arange(S2, dtype=torch.int32, device="cuda").expand(1, S1, 1, S2).contiguous()
    d_values = torch.randn((1, S1, 1, S2), generator=g, device="cuda")
    dq, dk, dw = dsa.lightning_indexer_bwd_raw(query, key, weights, indices, d_values)
    keys, want_k = key[0, :, 0].double(), torch.zeros((S2, 128), dtype=torch.float64, device="cuda")
    for s in range(0, S1, 5000):
        q, gr, w = query[0, s:s + 5000].double(), d_values[0, s:s + 5000, 0].double(), weights[0, s:s + 5000].double()
        z = q @ keys.T
        want_w = (z.clamp(min=0) * gr[:, None]).sum(2)
        dz = (z > 0) * gr[:, None] * w[:, :, None]
        want_q = dz @ keys
        want_k += torch.einsum("shk,shd->kd", dz, q)
        assert float((dq[0, s:s + 5000].double() - want_q).norm() / want_q.norm()) <= 2 * 2.0 ** -8
        assert float((dw[0, s:s + 5000].double() - want_w).norm() / want_w.norm()) <= 2.0 ** -18
    # dz rounded once, of every term
    assert float((dk[0, :, 0].double() - want_k).norm() / want_k.norm()) <= 2.0 ** -8
    check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["query", "key", "weights"])
def test_unlisted_values_whose_products_overflow(where):
    """Finite, but with infinite products: rows that take part in no listed pair leave the gradients as they are."""
    g = torch.Generator().manual_seed(29)
    B, S1, S2, N1, K = 1, 1501, 1280, 32, 1279
    query, key, weights, _ = (t.cuda() for t in make_indexer(g, B, S1, S2, N1, 4, torch.bfloat16))
    indices = torch.arange(K, dtype=torch.int32).expand(B, S1, 1, K).clone()   # not key 1279
    indices[0, 40] = -1
    indices = indices.cuda()
    d_values = torch.randn(indices.shape, generator=g).cuda() * 1e-3
    want = dsa.lightning_indexer_bwd_raw(query, key, weights, indices, d_values)
    if where == "query":
        query[0, 40] = 3e38
    elif where == "key":
        key[0, S2 - 1] = -3e38
    else:
        weights[0, 40] = 3e38
    got = dsa.lightning_indexer_bwd_raw(query, key, weights, indices, d_values)
    # (two kernels' gradients: each within the bounds of the test above)
    for name, a, b, bound in zip("qkw", got, want, (4 * 2.0 ** -8, 2 * 2.0 ** -8, 2 * 2.0 ** -18)):
        assert bool(torch.isfinite(a.float()).all()) and relative(a, b.cpu().double()) <= bound, f"d{name}"
    assert not got[0][0, 40].any() and not got[2][0, 40].any() and not got[1][0, S2 - 1].any()
    check_status()


@pytest.mark.gpu
def test_a_key_listed_twice_counts_twice():
    g = torch.Generator().manual_seed(11)
    query, key, weights, indices = make_indexer(g, 1, 3, 200, 64, 64, torch.bfloat16)
    indices[0, :, 0, 3] = indices[0, :, 0, 60]
    d_values = torch.randn(indices.shape, generator=g)
    dq, dk, dw = dsa.lightning_indexer_bwd_raw(query.cuda(), key.cuda(), weights.cuda(), indices.cuda(), d_values.cuda())
    want, err = indexer_gradients(query, key, weights, indices, d_values.masked_fill(indices < 0, 0.0))
    for name, got in (("q", dq), ("k", dk), ("w", dw)):
        assert bool(((got.cpu().double() - want[name]).abs() <= err[name] + want[name].abs() * 2.0 ** -7 + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,S1,S2,N1,K", [(2, 5, 60, 7, 40), (1, 1501, 1280, 32, 1279)])
def test_gradients_into_rows_of_any_alignment(B, S1, S2, N1, K, dtype):
    """d_q of the C entry need only start at an element, queries without keys included; the elements around it stay as they are."""
    from tilelang_ascend_b200 import _lib
    g = torch.Generator().manual_seed(33)
    query, key, weights, _ = (t.cuda() for t in make_indexer(g, B, S1, S2, N1, 4, dtype))
    indices = torch.arange(K, dtype=torch.int32).expand(B, S1, 1, K).clone()
    indices[0, 1], indices[-1, S1 - 1] = -1, -1
    indices, d_values = indices.cuda(), torch.randn((B, S1, 1, K), generator=g).cuda()
    sizes = B, S1, S2, N1, 128, K, _lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_FP16
    lib = _lib.load()
    nbytes = lib.dsa_lightning_indexer_bwd_workspace_bytes(*sizes)
    workspace = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
    want = indexer_gradients(query.cpu(), key.cpu(), weights.cpu(), indices.cpu(), d_values.cpu())[0]["q"] if S1 < 100 else dsa.lightning_indexer_bwd_raw(
        query, key, weights, indices, d_values)[0].cpu().double()
    for offset in (1, 4):
        buffer = torch.full((query.numel() + 8,), 7.0, dtype=dtype, device="cuda")
        d_q = buffer[offset:offset + query.numel()].view(query.shape)
        d_k, d_w = torch.zeros(key.shape, device="cuda"), torch.empty_like(weights)
        _lib.check(lib.dsa_lightning_indexer_bwd(query.data_ptr(), key.data_ptr(), weights.data_ptr(), indices.data_ptr(), d_values.data_ptr(), d_q.data_ptr(),
                                                 d_k.data_ptr(), d_w.data_ptr(), *sizes, workspace.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream))
        check_status()
        # dz rounded once and the result once, on either side
        assert relative(d_q, want) <= 4 * HALF_STEP[dtype]
        assert not d_q[0, 1].any() and not d_q[-1, S1 - 1].any() and not d_w[0, 1].any()
        assert bool((buffer[:offset] == 7).all()) and bool((buffer[offset + query.numel():] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("level", [2.0 ** 8, 2.0 ** -60, 2.0 ** 90])
def test_fp16_gradients_far_below_a_lists_largest(level):
    """fp16: heads with small weights and keys with small gradients, 2^-22 of the list's largest, keep the digits of one rounding."""
    g = torch.Generator().manual_seed(41)
    B, S1, S2, N1, K = 1, 6, 300, 64, 200
    query, key, _, indices = make_indexer(g, B, S1, S2, N1, K, torch.float16)
    small_head, small_key = torch.arange(N1) % 2 == 1, torch.arange(S2) >= S2 // 2

    def spread(shape):   # of either sign, from 1/2 to 1
        return (0.5 + 0.5 * torch.rand(shape, generator=g)) * torch.where(torch.rand(shape, generator=g) < 0.5, -1.0, 1.0)

    weights = spread((B, S1, N1)) * torch.where(small_head, 2.0 ** -22, 1.0)
    d_values = spread(indices.shape) * torch.where(small_key[indices.clamp(0, S2 - 1).long()], 2.0 ** -22, 1.0)
    if level < 1:
        weights = weights * level          # (both factors far from 1, their product times the queries and keys inside fp16)
        d_values = d_values * (2.0 ** 8 / level)
    else:
        weights = weights * (2.0 ** 8 / level)
        d_values = d_values * level
    dq, dk, dw = dsa.lightning_indexer_bwd_raw(query.cuda(), key.cuda(), weights.cuda(), indices.cuda(), d_values.cuda())
    check_status()
    want_q, want_k, err_q, err_k = (torch.zeros(t.shape, dtype=torch.float64) for t in (query, key, query, key))
    for s in range(S1):
        idx = indices[0, s, 0].long()
        there = (idx >= 0) & (idx < S2)
        idx, gr = idx[there], d_values[0, s, 0][there].double()
        rows, heads, w = key[0, idx, 0].double(), query[0, s].double(), weights[0, s].double()
        dz = torch.where(rows @ heads.T > 0, gr[:, None] * w, 0.0)
        # a half step of fp16 (and of fp32 for its factors), half a step of its smallest values below 2^-27 of the largest; sums in fp32
        top = float(gr.abs().max() * w.abs().max()) if gr.numel() else 0.0
        off = dz.abs() * (2.0 ** -11 + 2.0 ** -16) + 2.0 ** -38 * top
        want_q[0, s], err_q[0, s] = dz.T @ rows, off.T @ rows.abs()
        want_k[0, :, 0].index_add_(0, idx, dz @ heads)
        err_k[0, :, 0].index_add_(0, idx, off @ heads.abs())
    off_q = (dq.cpu().double() - want_q).abs()
    assert bool((off_q <= err_q + (want_q.abs() + err_q) * 2.0 ** -11 + 2.0 ** -25).all()), f"dq off, of small heads by {relative(dq[0, :, small_head.cuda()], want_q[0, :, small_head]):.3g}"
    off_k = (dk.cpu().double() - want_k).abs()
    assert bool((off_k <= err_k).all()), f"dk off, of small keys by {relative(dk[0, small_key.cuda()], want_k[0, small_key]):.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_are_not_finite_reach_the_gradients(dtype):
    """NaN and infinities among listed queries and keys: NaN where autograd through the definition has them, the same values elsewhere; entries that take no
    part stay out."""
    g = torch.Generator().manual_seed(43)
    B, S1, S2, N1, K = 1, 9, 300, 40, 150
    query, key, weights, indices = make_indexer(g, B, S1, S2, N1, K, dtype)
    clean = [t.clone() for t in (query, key)]
    query[0, 2, 3, 5], query[0, 4, 6, 7] = float("nan"), INF
    key[0, 7, 0, 9], key[0, 9, 0, 11] = float("nan"), -INF
    indices[0, :, 0][(indices[0, :, 0] == 7) | (indices[0, :, 0] == 9)] = -1
    indices[0, 6, 0, 100], indices[0, 7, 0, 20] = 7, 9      # one query lists each of them
    d_values = torch.randn(indices.shape, generator=g)
    d_values[indices < 0] = float("nan")
    got = [t.cpu().double() for t in dsa.lightning_indexer_bwd_raw(query.cuda(), key.cuda(), weights.cuda(), indices.cuda(), d_values.cuda())]
    check_status()

    def definition(query, key):
        leaves = [t.double().requires_grad_() for t in (query, key, weights)]
        total = 0.0
        for s in range(S1):
            idx = indices[0, s, 0].long()
            there = (idx >= 0) & (idx < S2)
            scores = (leaves[1][0, idx[there], 0] @ leaves[0][0, s].T).relu() @ leaves[2][0, s]
            total = total + (scores * d_values[0, s, 0][there].double()).sum()
        return torch.autograd.grad(total, leaves)

    want = definition(query, key)
    sizes = definition(*clean)
    for name, a, b, c in zip("qkw", got, want, sizes):
        assert torch.equal(a.isnan(), b.isnan()), f"d{name}: {int(a.isnan().sum())} values are NaN, of {int(b.isnan().sum())}"
        there = b.isfinite()
        assert torch.equal(a[~there].nan_to_num(0.0), b[~there].nan_to_num(0.0)), f"d{name}: infinities"
        # dz rounded once, the result once
        off = float((a - b)[there].norm() / c.norm())
        assert off <= 2 * HALF_STEP[dtype], f"d{name} off by {off:.3g} of its norm"
    assert bool(want[2][0, 2, 3].isnan()) and bool(want[2][0, 6].isnan().all()) and int(want[2].isnan().sum()) < 3 * N1


# ------------------------------------------------------------------------------------------------------ distillation
@pytest.mark.gpu
@pytest.mark.parametrize("kind,T", [("weights", 1.0), ("logits", 2.0)])
def test_distillation_through_the_indexer(kind, T):
    """Loss and gradients against autograd through the definition, from the indexer's own lists and scores."""
    g = torch.Generator().manual_seed(6)
    B, S1, S2, N1, K = 2, 9, 120, 64, 64
    query, key, weights, _ = make_indexer(g, B, S1, S2, N1, K, torch.bfloat16)
    leaves = [t.cuda().requires_grad_() for t in (query, key, weights)]
    indices, values = dsa.lightning_indexer_raw(*[t.detach() for t in leaves], sparse_count=K, sparse_mode=3, return_value=True)
    teacher = torch.randn(indices.shape, generator=g)
    teacher = (teacher.exp() if kind == "weights" else teacher).masked_fill(indices.cpu() < 0, float("nan"))
    up = torch.rand((B, S1), generator=g)
    loss = dsa.lightning_indexer_distillation(*leaves, indices, values, teacher.cuda(), teacher_kind=kind, temperature=T)
    loss.backward(up.cuda())
    check_status()
    qd, kd, wd = (t.double().requires_grad_() for t in (query, key, weights))
    ref = torch.zeros(B, S1, dtype=torch.float64)
    parts = []
    for b in range(B):
        for s in range(S1):
            idx = indices[b, s, 0].cpu().long()
            t = teacher[b, s, 0][idx >= 0].double()
            idx = idx[idx >= 0]
            scores = ((kd[b, idx, 0] @ qd[b, s].T).relu() @ wd[b, s]) / T
            p = t / t.sum() if kind == "weights" else torch.softmax(t / T, 0)
            parts.append((p * (p.log() - torch.log_softmax(scores, 0))).sum())
            ref[b, s] = parts[-1].detach()
    grads = torch.autograd.grad((torch.stack(parts) * up.double().flatten()).sum(), (qd, kd, wd))
    assert loss.shape == (B, S1) and float((loss.detach().cpu().double() - ref).abs().max()) < 1e-5
    # bf16: one rounding of each dz and one of the result; the fp32 gradient of the scores adds 2^-20
    for leaf, want, steps in zip(leaves, grads, (2 * 2.0 ** -8, 2 * 2.0 ** -8, 2.0 ** -16)):
        assert leaf.grad.dtype == leaf.dtype
        assert float((leaf.grad.cpu().double() - want).norm()) <= steps * float(want.norm())


@pytest.mark.gpu
def test_training_step_of_an_indexer():
    """The operators as a training step runs them: norm and rotation of both paths' queries and keys, indexer, attention on its lists,
    teacher, distillation, and the gradient back to the rows before the norm."""
    g = torch.Generator().manual_seed(12)
    B, S, H, K = 2, 160, 16, 64
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
    positions = torch.arange(S, dtype=torch.int32).repeat(B, 1).cuda()
    raw = {n: torch.randn(shape, generator=g).to(torch.bfloat16).cuda().requires_grad_() for n, shape in
           (("q", (B, S, H, 576)), ("kv", (B, S, 1, 576)), ("qi", (B, S, 64, 128)), ("ki", (B, S, 1, 128)))}
    ln_w, ln_b = torch.ones(128, device="cuda", requires_grad=True), torch.zeros(128, device="cuda", requires_grad=True)
    head_w = (torch.randn((B, S, 64), generator=g) / 512).cuda().requires_grad_()

    def forward():
        q, kv = dsa.qk_norm_rope(raw["q"], raw["kv"], positions, inv_freq, rope_start=512, k_norm="rms", norm_dim=512)
        qi, ki = dsa.qk_norm_rope(raw["qi"], raw["ki"], positions, inv_freq, interleaved=False, k_norm="layer", k_weight=ln_w, k_bias=ln_b)
        indices, values = dsa.lightning_indexer_raw(qi.detach(), ki.detach(), head_w.detach(), sparse_count=K, sparse_mode=3, return_value=True)
        out, lse = dsa.sparse_mla(q, kv, indices)
        teacher = dsa.sparse_mla_key_weights(q.detach(), kv.detach(), indices, lse)
        return qi, ki, indices, values, teacher, out, dsa.lightning_indexer_distillation(qi, ki, head_w, indices, values, teacher)

    qi, ki, indices, values, teacher, out, loss = forward()
    (loss.mean() + out.float().square().mean()).backward()
    check_status()
    assert bool(torch.isfinite(loss).all()) and bool((loss >= -1e-6).all())
    assert all(bool(torch.isfinite(t.grad).all()) and bool(t.grad.any()) for t in (*raw.values(), ln_w, ln_b, head_w))
    # the distillation's part, from the same rounded rows, lists, scores and teacher: gradients of qi and ki in 64 bits, then through the
    # norm and rotation by the operator's own (tested) backward
    p = teacher.double() / teacher.double().sum(-1, keepdim=True)
    soft = torch.softmax(values.double(), -1)
    d_values = ((soft - p) / (B * S)).masked_fill(indices < 0, 0.0).cpu()
    want, _ = indexer_gradients(qi.detach().cpu(), ki.detach().cpu(), head_w.detach().cpu(), indices.cpu(), d_values)
    dx = dsa.qk_norm_rope_bwd_raw(want["q"].to(torch.bfloat16).cuda(), None, None, None, positions, inv_freq, interleaved=False)[0]
    # dz, the result, and the rows behind the rotation are rounded once each on either side
    assert float((raw["qi"].grad.double() - dx.double()).norm()) <= 4 * 2.0 ** -8 * float(dx.double().norm())
    _, dk, _, _, dlw, dlb = dsa.qk_norm_rope_bwd_raw(None, want["k"].to(torch.bfloat16).cuda(), None, raw["ki"].detach(), positions, inv_freq,
                                                     interleaved=False, k_norm="layer", k_weight=ln_w.detach(), k_bias=ln_b.detach())
    for got, ref in ((raw["ki"].grad, dk), (ln_w.grad, dlw), (ln_b.grad, dlb)):
        assert float((got.double() - ref.double()).norm()) <= 4 * 2.0 ** -8 * float(ref.double().norm())
    assert float((head_w.grad.cpu().double() - want["w"]).norm()) <= 2.0 ** -12 * float(want["w"].norm())


@pytest.mark.gpu
def test_serving_step_reads_the_rows_it_wrote():
    """Decode: the step's latent and index keys go to the paged caches, the indexer and the attention read them from there."""
    g = torch.Generator().manual_seed(13)
    B, H, K, bs, blocks = 3, 16, 64, 16, 8
    lengths = torch.tensor([100, 65, 128])
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32)
    dt = torch.bfloat16
    latent, rope, keys = (torch.randn((B * blocks, bs, 1, d), generator=g).to(dt).cuda() for d in (512, 64, 128))
    q, kv, qi, ki = (torch.randn((B, 1, h, d), generator=g).to(dt).cuda() for h, d in ((H, 576), (1, 576), (64, 128), (1, 128)))
    w = (torch.rand((B, 1, 64), generator=g) / 64).cuda()
    last = lengths - 1
    slots = (table[torch.arange(B), last // bs] * bs + last % bs).view(B, 1).to(torch.int32)
    inv_freq = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
    pos = last.view(B, 1).to(torch.int32).cuda()
    kw = dict(rope_start=512, k_norm="rms", norm_dim=512)
    old = latent.clone()
    qr = dsa.qk_norm_rope_cached(q, kv, pos, inv_freq, latent, slots.cuda(), key_cache_rope=rope, **kw)
    qir = dsa.qk_norm_rope_cached(qi, ki, pos, inv_freq, keys, slots.cuda(), interleaved=False, k_norm="layer")
    idx, _ = dsa.lightning_indexer(qir, keys, w, actual_seq_lengths_key=lengths.to(torch.int32), block_table=table.cuda(), layout_key="PA_BSND", sparse_count=K)
    out = dsa.sparse_attn_tilelang(qr[..., :512].contiguous(), latent, latent, idx, 576 ** -0.5, 1, torch.ones(B, dtype=torch.int32), lengths,
                                   query_rope=qr[..., 512:].contiguous(), key_rope=rope, layout_kv="PA_BSND", block_table=table.cuda())
    check_status()
    assert int((latent != old).any(-1).sum()) == B
    # dense copies of the caches give the same lists and rows
    rows = (table.long()[:, :, None] * bs + torch.arange(bs)).view(B, -1).cuda()
    for b in range(B):
        n = int(lengths[b])
        kd = keys.view(-1, 128)[rows[b, :n]].view(1, n, 1, 128)
        idx_d, _ = dsa.lightning_indexer(qir[b:b + 1], kd, w[b:b + 1], sparse_count=K)
        assert torch.equal(idx_d[0], idx[b])
        kvd = torch.cat((latent.view(-1, 512)[rows[b, :n]], rope.view(-1, 64)[rows[b, :n]]), -1).view(1, n, 1, 576)
        out_d, _ = dsa.sparse_mla_fwd_raw(qr[b:b + 1], kvd, idx_d, sm_scale=576 ** -0.5, q_start=n - 1, causal=True, dv=512)
        assert float((out_d - out[b:b + 1]).float().abs().max()) <= 2.0 ** -7
        # the row written last is the normed and rotated one
        direct = dsa.qk_norm_rope(None, kv[b:b + 1], pos[b:b + 1], inv_freq, **kw)[1]
        assert torch.equal(direct[0, 0, 0], kvd[0, n - 1, 0])


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(14)
    query, key, weights, indices = (t.cuda() for t in make_indexer(g, 1, 20, 400, 64, 128, torch.bfloat16))
    q, kv = torch.randn((1, 20, 128, 576), generator=g).to(torch.bfloat16).cuda(), torch.randn((1, 400, 1, 576), generator=g).to(torch.bfloat16).cuda()
    lse = torch.randn((1, 20, 128), generator=g).cuda() + 6
    d_values = torch.randn(indices.shape, generator=g).cuda()

    def step():
        return (dsa.sparse_mla_key_weights(q, kv, indices, lse),) + dsa.lightning_indexer_bwd_raw(query, key, weights, indices, d_values)

    def same(a, b):   # (d_key: the order of its additions is free; the others are repeatable)
        return all(torch.equal(x, y) for x, y in zip((a[0], a[1], a[3]), (b[0], b[1], b[3]))) and torch.allclose(a[2], b[2], rtol=1e-4, atol=1e-5)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.synchronize()
    assert same(first, step()) and same(first, other)
    q.mul_(0.5)
    d_values.mul_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert same(captured, step())
    graph.replay()
    torch.cuda.synchronize()
    assert same(captured, step())
    check_status()


@pytest.mark.gpu
def test_calls_at_the_same_time_and_two_graphs():
    """Calls that overlap on two streams, and two graphs of one call replayed in turn, do not touch one another's results: sizes that take each of the two
    ways through the indexer's backward."""
    g = torch.Generator().manual_seed(15)
    small = [t.cuda() for t in make_indexer(g, 2, 60, 500, 64, 200, torch.bfloat16)]
    large = [t.cuda() for t in make_indexer(g, 1, 1500, 1500, 16, 1400, torch.bfloat16)]
    grads = [torch.randn(s[3].shape, generator=g).cuda() for s in (small, large)]
    q, kv = torch.randn((1, 300, 128, 576), generator=g).to(torch.bfloat16).cuda(), torch.randn((1, 700, 1, 576), generator=g).to(torch.bfloat16).cuda()
    idx, lse = lists(g, 1, 300, 700, 300).cuda(), torch.randn((1, 300, 128), generator=g).cuda() + 6

    def step(which):
        dq, dk, dw = dsa.lightning_indexer_bwd_raw(*(small, large)[which], grads[which])
        return dq, dw, dsa.sparse_mla_key_weights(q, kv, idx, lse)

    want = [step(0), step(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, captured = [], []
    for i, stream in enumerate(streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                captured.append(step(i))
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(3):
        got = [None, None]
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = step(i)
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])) and all(torch.equal(a, b) for a, b in zip(captured[i], want[i]))
    check_status()


@pytest.mark.gpu
def test_a_whole_step_in_a_graph():
    """Forward and backward of the distillation through autograd, captured and replayed on other inputs."""
    g = torch.Generator().manual_seed(16)
    query, key, weights, _ = make_indexer(g, 1, 1500, 1500, 16, 4, torch.bfloat16)
    leaves = [t.cuda().requires_grad_() for t in (query, key, weights)]
    indices, values = dsa.lightning_indexer_raw(*[t.detach() for t in leaves], sparse_count=1400, sparse_mode=3, return_value=True)
    teacher = torch.rand(indices.shape, generator=g).cuda()

    def step():
        loss = dsa.lightning_indexer_distillation(*leaves, indices, values, teacher)
        return (loss.detach(),) + torch.autograd.grad(loss.sum(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.synchronize()
    teacher.copy_(torch.rand(indices.shape, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    again = step()
    assert all(torch.equal(captured[i], again[i]) for i in (0, 1, 3)) and relative(captured[2], again[2].cpu().double()) < 2.0 ** -7
    check_status()


@pytest.mark.gpu
def test_weights_of_any_alignment_and_other_head_counts():
    """Head weights off a 16-byte boundary, and 48 heads, where the lists hold most keys."""
    g = torch.Generator().manual_seed(17)
    for N1, offset in ((32, 1), (48, 0)):
        query, key, weights, indices = (t.cuda() for t in make_indexer(g, 2, 1030, 1290, N1, 700, torch.bfloat16))
        buffer = torch.zeros(weights.numel() + 4, device="cuda")
        moved = buffer[offset:offset + weights.numel()].view(weights.shape)
        moved.copy_(weights)
        d_values = torch.randn(indices.shape, generator=g).cuda()
        dq, dk, dw = dsa.lightning_indexer_bwd_raw(query, key, moved, indices, d_values)
        # the same through fp16, whose gradient always takes the other way (values of eight bits are exact in both types)
        hq, hk, hw = dsa.lightning_indexer_bwd_raw(query.half(), key.half(), weights, indices, d_values)
        for got, ref, bound in ((dq, hq, 2 * 2.0 ** -8), (dk, hk, 2 * 2.0 ** -8), (dw, hw, 2.0 ** -18)):
            assert relative(got, ref.cpu().double()) <= bound
    check_status()


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    q, kv = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 9, 1, 64, dtype=torch.bfloat16)
    idx, lse = torch.zeros(1, 2, 1, 8, dtype=torch.int32), torch.zeros(1, 2, 4)
    qi, ki, w = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16), torch.zeros(1, 9, 1, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 4)
    val = torch.zeros(1, 2, 1, 8)
    distil = dsa.lightning_indexer_distillation
    bad = [
        lambda: dsa.sparse_mla_key_weights(q[0], kv, idx, lse),
        lambda: dsa.sparse_mla_key_weights(q.float(), kv.float(), idx, lse),
        lambda: dsa.sparse_mla_key_weights(q, kv[..., :32], idx, lse),
        lambda: dsa.sparse_mla_key_weights(q, kv, idx[:, :1], lse),
        lambda: dsa.sparse_mla_key_weights(q, kv, idx, lse[:, :, :3]),
        lambda: dsa.sparse_mla_key_weights(q[..., :60].contiguous(), kv[..., :60].contiguous(), idx, lse),
        lambda: dsa.sparse_mla_key_weights(q, kv, idx.long(), lse),
        lambda: dsa.sparse_mla_key_weights(q, kv.half(), idx, lse),
        lambda: dsa.sparse_mla_key_weights(q, kv, idx, lse.double()),
        lambda: dsa.sparse_mla_key_weights(q, kv, torch.zeros(1, 2, 1, 8193, dtype=torch.int32), lse),
        lambda: dsa.sparse_mla_key_weights(q, kv, idx[..., :0], lse),
        lambda: dsa.lightning_indexer_bwd_raw(qi[..., :64], ki[..., :64], w, idx, val),
        lambda: dsa.lightning_indexer_bwd_raw(torch.zeros(1, 2, 65, 128, dtype=torch.bfloat16), ki, torch.zeros(1, 2, 65), idx, val),
        lambda: dsa.lightning_indexer_bwd_raw(qi, ki, w.bfloat16(), idx, val),
        lambda: dsa.lightning_indexer_bwd_raw(qi, ki, w, idx, val.bfloat16()),
        lambda: dsa.lightning_indexer_bwd_raw(qi, ki, w, idx, val[..., :4]),
        lambda: dsa.lightning_indexer_bwd_raw(qi, ki.half(), w, idx, val),
        lambda: dsa.lightning_indexer_bwd_raw(qi.transpose(1, 2), ki, w.transpose(1, 2), idx[:, :1].expand(1, 4, 1, 8), val[:, :1].expand(1, 4, 1, 8)),
        lambda: distil(qi, ki, w, idx, val, val[:, :1]),
        lambda: distil(qi, ki, w, idx, val.half(), val),
        lambda: distil(qi, ki, w, idx[:, :, 0], val, val),
    ]
    for call in bad:
        with pytest.raises(ValueError) as e:
            call()
        assert "no CPU path" not in str(e.value), str(e.value)
    for call in (lambda: dsa.sparse_mla_key_weights(q, kv, idx, lse), lambda: dsa.lightning_indexer_bwd_raw(qi, ki, w, idx, val), lambda: distil(qi, ki, w, idx, val, val),
                 ):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_c_entries_refuse_before_any_cuda_call():
    from tilelang_ascend_b200 import _lib
    lib = _lib.load()
    assert lib.dsa_sparse_mla_key_weights(None, None, None, None, None, 1, 1, 1, 1, 64, 8, 1.0, 0, 1, 0, None) != 0
    assert lib.dsa_lightning_indexer_bwd(None, None, None, None, None, None, None, None, 1, 1, 1, 1, 128, 8, 0, None, 0, None) != 0
