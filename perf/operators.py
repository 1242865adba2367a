"""Performance cases of the operators around the sparse-attention path: the per-head norm with rotation that makes its queries
and keys (and fills its paged key caches), the attention weights of the listed keys, and the distillation that trains the
lightning indexer with them.

Kinds (each is one public call, or one forward + backward):

* ``cache``    norm + rotation of a step's queries and latent keys, keys written to a paged cache (``qk_norm_rope_cached``)
* ``rope``     differentiable norm + rotation of queries and keys, forward and backward (``qk_norm_rope`` + autograd)
* ``weights``  head-averaged attention weights of the listed keys (``sparse_mla_key_weights``)
* ``distill``  distillation of a row of logits from a teacher's top entries, forward and backward (``topk_distillation``)
* ``indexer``  the same through the lightning indexer: loss, and gradients of its queries, keys and head weights
               (``lightning_indexer_distillation``)

``own`` selects the package's kernels; otherwise ``run`` computes the same in elementary torch operations.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 128        # rows per block of the paged caches
_EPS = 1e-6
_ID = 128           # dims of the indexer's queries and keys


def listed():
    return [
        # decode step of a full batch: 128 heads of 512 + 64 dims, latent keys into a cache kept in two parts
        dict(name="cache_decode_64", kind="cache", B=64, S=1, H=128, D=576, R=64, dtype="bf16", parts=2, interleaved=True),
        # the same for a 4096-token prompt chunk
        dict(name="cache_prefill_4096", kind="cache", B=1, S=4096, H=128, D=576, R=64, dtype="bf16", parts=2, interleaved=True),
        # one training step of the indexer's 64 query heads and its layer-normed key, the first 64 dims rotated
        dict(name="rope_train_indexer_4096", kind="rope", B=1, S=4096, H=64, HK=1, D=128, R=64, start=0, q_norm="none", k_norm="layer",
             dtype="bf16", interleaved=False),
        # ragged batch of a tensor-parallel share of heads, every query and key head RMS-normed, slices of one projection, fp16
        dict(name="rope_train_3x333_fp16", kind="rope", B=3, S=333, H=16, HK=4, D=128, R=128, start=0, q_norm="rms", k_norm="rms",
             dtype="fp16", interleaved=False),
        # the teacher of one layer's indexer at the prefill shape: 4096 queries, 128 heads, top-2048
        dict(name="weights_4096", kind="weights", B=1, S=4096, S_kv=4096, H=128, topk=2048, dtype="bf16"),
        # two ragged sequences on half of the heads, shorter lists, fp16
        dict(name="weights_2x333_h64_fp16", kind="weights", B=2, S=333, S_kv=2501, H=64, topk=1024, dtype="fp16"),
        # a short list for a few queries: latency
        dict(name="distill_list_16x512", kind="distill", rows=16, V=512, K=512, over="list", teacher_kind="weights", T=1.0, dtype="fp32"),
        # every query's list of the prefill shape
        dict(name="distill_list_4096x2048", kind="distill", rows=4096, V=2048, K=2048, over="list", teacher_kind="weights", T=1.0, dtype="fp32"),
        # scores against a whole 128 K context, the teacher's top 2048 of each row, normalised over the row
        dict(name="distill_row_1024x131072", kind="distill", rows=1024, V=131072, K=2048, over="row", teacher_kind="logits", T=2.0, dtype="fp32"),
        # the indexer's training step at the prefill shape: 64 heads, top-2048 of 4096 keys
        dict(name="indexer_4096", kind="indexer", B=1, S=4096, S_kv=4096, H=64, topk=2048, dtype="bf16"),
        # two ragged sequences, 32 heads, short lists, fp16
        dict(name="indexer_2x301_h32_fp16", kind="indexer", B=2, S=301, S_kv=1507, H=32, topk=512, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; odd ones as likely as even ones."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["cache", "rope", "weights", "distill", "indexer"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "cache":
        H = rng.choice([16, 32, 64, 128])
        if rng.random() < 0.5:
            return dict(kind=kind, B=_log(rng, 1, 256), S=rng.choice([1, 1, 2]), H=H, D=576, R=64, dtype=dtype, parts=rng.choice([1, 2]),
                        interleaved=rng.random() < 0.5)
        return dict(kind=kind, B=rng.choice([1, 1, 2]), S=_log(rng, 16, 2048), H=H, D=576, R=64, dtype=dtype, parts=rng.choice([1, 2]),
                    interleaved=rng.random() < 0.5)
    if kind == "rope":
        D, R, start = rng.choice([(128, 64, 0), (128, 128, 0), (576, 64, 512), (192, 64, 128), (64, 64, 0), (256, 64, 192)])
        HK = rng.choice([1, 1, 2, 8])
        return dict(kind=kind, B=rng.choice([1, 2, 3]), S=_log(rng, 1, 1365), H=HK * rng.choice([4, 8, 16]), HK=HK, D=D, R=R, start=start,
                    q_norm=rng.choice(["none", "rms"]), k_norm=rng.choice(["rms", "layer"]), dtype=dtype, interleaved=rng.random() < 0.5)
    if kind == "weights":
        S = _log(rng, 1, 2048)
        return dict(kind=kind, B=rng.choice([1, 1, 2]), S=S, S_kv=_log(rng, max(S, 64), 8192), H=rng.choice([16, 64, 128, 128]),
                    topk=rng.choice([256, 512, 1024, 2048]), dtype=dtype)
    if kind == "distill":
        teacher_kind, T = rng.choice(["weights", "logits"]), rng.choice([1.0, 1.0, 2.0])
        if rng.random() < 0.5:
            K = _log(rng, 64, 4096)
            return dict(kind=kind, rows=_log(rng, 1, 4096), V=K, K=K, over="list", teacher_kind=teacher_kind, T=T, dtype=rng.choice(["fp32", "fp32", dtype]))
        V = _log(rng, 1000, 131072)
        return dict(kind=kind, rows=_log(rng, 1, min(4096, (1 << 27) // V)), V=V, K=min(V, rng.choice([64, 512, 2048])), over=rng.choice(["row", "row", "list"]),
                    teacher_kind=teacher_kind, T=T, dtype=rng.choice(["fp32", dtype]))
    S = _log(rng, 1, 2048)
    return dict(kind=kind, B=rng.choice([1, 1, 2]), S=S, S_kv=_log(rng, max(S, 64), 8192), H=rng.choice([8, 16, 32, 64, 64]),
                topk=rng.choice([256, 512, 1024, 2048]), dtype=dtype)


# ----------------------------------------------------------------------------------------------------------- inputs
def _causal_lists(g, B, S, S_kv, topk, dev):
    """[B, S, 1, topk]: distinct keys in random order below each query's causal limit, -1 behind them."""
    limits = torch.arange(S, device=dev) + (S_kv - S + 1)
    out = torch.full((B, S, 1, topk), -1, dtype=torch.int32, device=dev)
    k = min(topk, S_kv)
    for b in range(B):
        keys = torch.rand((S, S_kv), generator=g, device=dev)
        keys = torch.where(torch.arange(S_kv, device=dev)[None, :] < limits[:, None], keys, torch.full_like(keys, -1.0))
        val, idx = keys.topk(k, dim=1)
        out[b, :, 0, :k] = torch.where(val < 0, torch.full_like(idx, -1), idx).to(torch.int32)
    return out


def _chunks(S, per_query_bytes):
    n = max(1, min(S, int((1 << 30) // max(1, per_query_bytes))))
    return [(s, min(S, s + n)) for s in range(0, S, n)]


def _attention_lse(q, kv, indices, scale):
    """Natural-log normaliser of every (query, head) over its list: what the attention's forward leaves behind."""
    B, S, H, D = q.shape
    K = indices.shape[3]
    lse = torch.empty((B, S, H), dtype=torch.float32, device=q.device)
    for b in range(B):
        for s0, s1 in _chunks(S, K * (D * 6 + H * 12)):
            idx = indices[b, s0:s1, 0].long()
            rows = kv[b, idx.clamp(min=0), 0].float()
            sc = torch.matmul(q[b, s0:s1].float(), rows.transpose(1, 2)) * scale
            sc.masked_fill_((idx < 0)[:, None, :], float("-inf"))
            lse[b, s0:s1] = torch.logsumexp(sc, dim=2)
    return lse


def _eight_bit(x):
    """Values as the indexer's 8-bit quantiser leaves them (steps of 1/16, +-8)."""
    return (x.float() * 16).round().clamp(-128, 127) / 16


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    c = dict(case)
    kind, dt = c["kind"], _DT[c["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    def weight(n):
        return (1 + 0.2 * randn(n, dtype=torch.float32)).to(dt)

    if kind in ("cache", "rope"):
        B, S, H, D, R = c["B"], c["S"], c["H"], c["D"], c["R"]
        s = dict(c)
        s["inv_freq"] = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().to(dev)
        first = torch.randint(0, 100000, (B, 1), generator=g, device=dev)
        s["positions"] = (first + torch.arange(S, device=dev)[None, :]).to(torch.int32).contiguous()
        if kind == "cache":
            s["start"] = D - R
            s["q"], s["k"], s["k_weight"] = randn(B, S, H, D), randn(B, S, 1, D), weight(D - R)
            blocks = 2 * (-(-B * S // _BLOCK)) + 1
            s["slots"] = torch.randperm(blocks * _BLOCK, generator=g, device=dev)[:B * S].to(torch.int32).view(B, S).contiguous()
            if c["parts"] == 2:
                s["cache"], s["cache_rope"] = randn(blocks, _BLOCK, 1, D - R), randn(blocks, _BLOCK, 1, R)
            else:
                s["cache"], s["cache_rope"] = randn(blocks, _BLOCK, 1, D), None
            return s
        HK = c["HK"]
        x = randn(B, S, (H + HK) * D)   # one projection's output; queries and keys are slices of it
        s["q"] = x[..., :H * D].view(B, S, H, D).detach().requires_grad_(True)
        s["k"] = x[..., H * D:].view(B, S, HK, D).detach().requires_grad_(True)
        s["norm_dim"] = c["start"] if c["start"] else D     # the rotated tail of a latent row is not normed
        s["grad_q"], s["grad_k"] = randn(B, S, H, D), randn(B, S, HK, D)
        for side in ("q", "k"):
            s[side + "_weight"] = weight(s["norm_dim"]).requires_grad_(True) if c[side + "_norm"] != "none" else None
            s[side + "_bias"] = (0.1 * randn(s["norm_dim"])).requires_grad_(True) if c[side + "_norm"] == "layer" else None
        return s
    if kind == "weights":
        B, S, S_kv, H = c["B"], c["S"], c["S_kv"], c["H"]
        s = dict(c, q=randn(B, S, H, 576), kv=randn(B, S_kv, 1, 576), indices=_causal_lists(g, B, S, S_kv, c["topk"], dev))
        s["lse"] = _attention_lse(s["q"], s["kv"], s["indices"], 576 ** -0.5)
        return s
    if kind == "distill":
        rows, V, K = c["rows"], c["V"], c["K"]
        student = (2.0 * randn(rows, V, dtype=torch.float32)).to(dt)
        indices = None
        if K < V:
            # distinct columns: a random start and a stride that shares no factor with the row's width
            stride = 2 * (V // (2 * K)) + 1
            while math.gcd(stride, V) != 1:
                stride += 2
            first = torch.randint(0, V, (rows, 1), generator=g, device=dev)
            indices = ((first + stride * torch.arange(K, device=dev)[None, :]) % V).to(torch.int32).contiguous()
        teacher = 2.0 * randn(rows, K, dtype=torch.float32)
        if c["teacher_kind"] == "weights":
            teacher = torch.softmax(teacher, dim=1)
        # causal rows: the last entries of early lists do not exist
        if indices is None:
            count = torch.randint(1, K + 1, (rows, 1), generator=g, device=dev)
            gone = torch.arange(K, device=dev)[None, :] >= torch.where(torch.rand((rows, 1), generator=g, device=dev) < 0.25, count, K)
            student = student.masked_fill(gone, float("-inf"))
        # the gradient of a mean over rows; of a scaled loss where the student's gradient is kept in fp16
        grad = torch.rand((rows,), generator=g, device=dev) * (4096.0 if c["dtype"] == "fp16" else 1.0 / rows)
        return dict(c, student=student.requires_grad_(True), teacher=teacher, indices=indices, grad=grad)
    B, S, S_kv, H, K = c["B"], c["S"], c["S_kv"], c["H"], c["topk"]
    s = dict(c, query=_eight_bit(randn(B, S, H, _ID)).to(dt), key=_eight_bit(randn(B, S_kv, 1, _ID)).to(dt),
             weights=randn(B, S, H, dtype=torch.float32) / (H * _ID ** 0.5), indices=_causal_lists(g, B, S, S_kv, K, dev))
    listed_keys = s["indices"] >= 0
    s["teacher"] = torch.softmax((2.0 * randn(B, S, 1, K, dtype=torch.float32)).masked_fill(~listed_keys, float("-inf")), dim=3)
    s["values"] = torch.full((B, S, 1, K), float("-inf"), dtype=torch.float32, device=dev)
    for b in range(B):
        for s0, s1 in _chunks(S, K * (_ID * 6 + H * 12)):
            _, _, _, z = _indexer_products(s, b, s0, s1)
            s["values"][b, s0:s1, 0] = (z.relu() * s["weights"][b, s0:s1, :, None]).sum(1)
    s["values"].masked_fill_(~listed_keys, float("-inf"))
    s["grad"] = torch.rand((B, S), generator=g, device=dev) * ((2.0 ** 20 if c["dtype"] == "fp16" else 1.0) / (B * S))   # fp16: of a scaled loss
    for name in ("query", "key", "weights"):
        s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _angles(s):
    angle = s["positions"].double()[..., None] * s["inv_freq"].double()
    return angle.cos().float()[:, :, None, :], angle.sin().float()[:, :, None, :]


def _pairs(x, interleaved):
    """The two members of every rotated pair."""
    if interleaved:
        return x[..., 0::2], x[..., 1::2]
    half = x.shape[-1] // 2
    return x[..., :half], x[..., half:]


def _unpairs(a, b, interleaved):
    return torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)


def _rotate(x, cos, sin, s):
    """Rotation of the dims [start, start + R) of fp32 rows."""
    r0, R = s["start"], s["R"]
    a, b = _pairs(x[..., r0:r0 + R], s["interleaved"])
    return torch.cat((x[..., :r0], _unpairs(a * cos - b * sin, b * cos + a * sin, s["interleaved"]), x[..., r0 + R:]), dim=-1)


def _norm(x, kind, n, weight, bias):
    """fp32 rows with their leading n dims normed; also the centred rows and the reciprocal deviation."""
    head = x[..., :n]
    if kind == "layer":
        head = head - head.mean(-1, keepdim=True)
    rstd = torch.rsqrt(head.square().mean(-1, keepdim=True) + _EPS)
    unit = head * rstd
    y = unit * weight.float()
    if bias is not None:
        y = y + bias.float()
    return torch.cat((y, x[..., n:]), dim=-1), unit, rstd


def _plain_cache(s):
    cos, sin = _angles(s)
    n = s["D"] - s["R"]
    q = _rotate(s["q"].float(), cos, sin, s).to(s["q"].dtype)
    k, _, _ = _norm(s["k"].float(), "rms", n, s["k_weight"], None)
    k = _rotate(k, cos, sin, s).to(s["k"].dtype)[:, :, 0].flatten(0, 1)
    rows = s["slots"].flatten().long()
    if s["cache_rope"] is None:
        s["cache"].view(-1, s["D"])[rows] = k
        return [q, s["cache"]]
    s["cache"].view(-1, n)[rows] = k[:, :n]
    s["cache_rope"].view(-1, s["R"])[rows] = k[:, n:]
    return [q, s["cache"], s["cache_rope"]]


def _plain_rope(s):
    cos, sin = _angles(s)
    n = s["norm_dim"]
    out = {}
    for side in ("q", "k"):
        x, kind, weight, bias = s[side].detach(), s[side + "_norm"], s[side + "_weight"], s[side + "_bias"]
        xf = x.float()
        if kind != "none":
            weight = weight.detach()
            xf, unit, rstd = _norm(xf, kind, n, weight, None if bias is None else bias.detach())
        out[side] = _rotate(xf, cos, sin, s).to(x.dtype)
        grad = _rotate(s["grad_" + side].float(), cos, -sin, s)
        if kind != "none":
            head = grad[..., :n]
            out["d_" + side + "_weight"] = (head * unit).sum((0, 1, 2)).to(weight.dtype)
            if bias is not None:
                out["d_" + side + "_bias"] = head.sum((0, 1, 2)).to(bias.dtype)
            head = head * weight.float()
            inner = head - unit * (head * unit).mean(-1, keepdim=True)
            if kind == "layer":
                inner = inner - head.mean(-1, keepdim=True)
            grad = torch.cat((inner * rstd, grad[..., n:]), dim=-1)
        out["d_" + side] = grad.to(x.dtype)
    return out


def _plain_weights(s):
    q, kv, indices = s["q"], s["kv"], s["indices"]
    B, S, H, D = q.shape
    K = indices.shape[3]
    out = torch.empty((B, S, 1, K), dtype=torch.float32, device=q.device)
    for b in range(B):
        for s0, s1 in _chunks(S, K * (D * 6 + H * 12)):
            idx = indices[b, s0:s1, 0].long()
            rows = kv[b, idx.clamp(min=0), 0].float()
            sc = torch.matmul(q[b, s0:s1].float(), rows.transpose(1, 2)) * D ** -0.5
            p = torch.exp(sc - s["lse"][b, s0:s1, :, None]).mean(1)
            out[b, s0:s1, 0] = p.masked_fill(idx < 0, 0.0)
    return out


def _teacher(teacher, kind, valid, T):
    if kind == "logits":
        t = (teacher / T).masked_fill(~valid, float("-inf"))
        p = torch.exp(t - t.amax(-1, keepdim=True))
    else:
        p = teacher.masked_fill(~valid, 0.0)
    return p / p.sum(-1, keepdim=True)


def _plain_distill(s):
    student, T = s["student"].detach(), s["T"]
    z = student.float() / T
    columns = None if s["indices"] is None else s["indices"].long()
    at = z if columns is None else z.gather(1, columns)
    valid = at > float("-inf")
    p = _teacher(s["teacher"], s["teacher_kind"], valid, T)
    norm = z if s["over"] == "row" else at
    top = norm.amax(-1, keepdim=True)
    e = torch.exp(norm - top)
    total = e.sum(-1, keepdim=True)
    log_s = at - top - torch.log(total)
    loss = torch.where(p > 0, p * (torch.log(p) - log_s), torch.zeros_like(p)).sum(-1)
    g = s["grad"][:, None] / T
    if columns is None:
        grad = g * (e / total - p)
    elif s["over"] == "row":
        grad = (g * (e / total)).scatter_add_(1, columns, -g * p)
    else:
        grad = torch.zeros_like(z).scatter_add_(1, columns, g * (e / total - p))
    return [loss, grad.to(student.dtype)]


def _indexer_products(s, b, s0, s1):
    """Queries, listed keys and head scores of queries [s0, s1) of a sequence; the 8-bit inputs make the products exact."""
    idx = s["indices"][b, s0:s1, 0].long()
    rows = s["key"].detach()[b, idx.clamp(min=0), 0].float()
    q = s["query"].detach()[b, s0:s1].float()
    return idx, q, rows, torch.matmul(q, rows.transpose(1, 2))


def _plain_indexer(s):
    query, key, weights = s["query"].detach(), s["key"].detach(), s["weights"].detach()
    B, S, H, _ = query.shape
    K = s["topk"]
    valid = s["values"] > float("-inf")
    p = _teacher(s["teacher"], "weights", valid, 1.0)
    top = s["values"].amax(-1, keepdim=True)
    e = torch.exp(s["values"] - top)
    total = e.sum(-1, keepdim=True)
    log_s = s["values"] - top - torch.log(total)
    loss = torch.where(p > 0, p * (torch.log(p) - log_s), torch.zeros_like(p)).sum((2, 3))
    d_values = s["grad"][:, :, None, None] * (e / total - p)
    d_query, d_weights = torch.empty_like(query), torch.empty_like(weights)
    d_key = torch.zeros(key.shape, dtype=torch.float32, device=key.device)
    for b in range(B):
        for s0, s1 in _chunks(S, K * (_ID * 10 + H * 16)):
            idx, q, rows, z = _indexer_products(s, b, s0, s1)
            dv = d_values[b, s0:s1, 0].masked_fill(idx < 0, 0.0)
            d_weights[b, s0:s1] = (z.relu() * dv[:, None, :]).sum(2)
            dz = (z > 0) * weights[b, s0:s1, :, None] * dv[:, None, :]
            d_query[b, s0:s1] = torch.matmul(dz, rows).to(query.dtype)
            d_key[b, :, 0].index_add_(0, idx.clamp(min=0).flatten(), torch.matmul(dz.transpose(1, 2), q).flatten(0, 1))
    return [loss, d_query, d_key.to(key.dtype), d_weights]


# --------------------------------------------------------------------------------------------------------- one pass
def run(s):
    kind = s["kind"]
    if not own:
        plain = {"cache": _plain_cache, "rope": _plain_rope, "weights": _plain_weights, "distill": _plain_distill, "indexer": _plain_indexer}
        return plain[kind](s)
    import tilelang_ascend_b200 as dsa
    if kind == "cache":
        q = dsa.qk_norm_rope_cached(s["q"], s["k"], s["positions"], s["inv_freq"], s["cache"], s["slots"], key_cache_rope=s["cache_rope"],
                                    rope_start=s["start"], interleaved=s["interleaved"], k_norm="rms", k_weight=s["k_weight"],
                                    norm_dim=s["D"] - s["R"], eps=_EPS)
        return [q, s["cache"]] + ([] if s["cache_rope"] is None else [s["cache_rope"]])
    if kind == "rope":
        norms = {side + "_norm": None if s[side + "_norm"] == "none" else s[side + "_norm"] for side in ("q", "k")}
        q, k = dsa.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], rope_start=s["start"], interleaved=s["interleaved"],
                                q_weight=s["q_weight"], q_bias=s["q_bias"], k_weight=s["k_weight"], k_bias=s["k_bias"], norm_dim=s["norm_dim"],
                                eps=_EPS, **norms)
        names = [n for n in ("q", "k", "q_weight", "q_bias", "k_weight", "k_bias") if s[n] is not None]
        grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["grad_q"], s["grad_k"]))
        return dict({"d_" + n: d for n, d in zip(names, grads)}, q=q.detach(), k=k.detach())
    if kind == "weights":
        return dsa.sparse_mla_key_weights(s["q"], s["kv"], s["indices"], s["lse"])
    if kind == "distill":
        loss = dsa.topk_distillation(s["student"], s["teacher"], s["indices"], teacher_kind=s["teacher_kind"], over=s["over"], temperature=s["T"])
        return [loss.detach(), *torch.autograd.grad(loss, s["student"], s["grad"])]
    loss = dsa.lightning_indexer_distillation(s["query"], s["key"], s["weights"], s["indices"], s["values"], s["teacher"])
    return [loss.detach(), *torch.autograd.grad(loss, (s["query"], s["key"], s["weights"]), s["grad"])]


# ------------------------------------------------------------------------------------------------------ what it takes
def work(case):
    c, kind = case, case["kind"]
    e = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
    if kind == "cache":
        T = c["B"] * c["S"]
        return {"bytes": 2 * T * (c["H"] + 1) * c["D"] * e + 8 * T, "flops": 6 * T * (c["H"] + 1) * c["D"]}
    if kind == "rope":
        n = c["B"] * c["S"] * (c["H"] + c["HK"]) * c["D"]
        return {"bytes": 4 * n * e + 4 * c["B"] * c["S"], "flops": 16 * n}
    if kind == "distill":
        rows, V, K = c["rows"], c["V"], c["K"]
        listed_bytes = rows * K * 4 * (2 if K < V else 1)
        read = rows * (V if c["over"] == "row" or K == V else K) * e
        return {"bytes": read + listed_bytes + rows * V * e + 8 * rows, "flops": 8 * rows * V}
    pairs = c["B"] * sum(min(c["topk"], c["S_kv"] - c["S"] + 1 + t) for t in range(c["S"]))
    B, S, S_kv, H, K = c["B"], c["S"], c["S_kv"], c["H"], c["topk"]
    if kind == "weights":
        return {"bytes": B * (S * H * (576 * e + 4) + S_kv * 576 * e + S * K * 8), "flops": 2 * 576 * H * pairs}
    return {"bytes": B * (2 * S * H * (_ID * e + 4) + 2 * S_kv * _ID * e + S * K * 12), "flops": 3 * 2 * _ID * H * pairs}


# ----------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """What ``run`` returns for these inputs, from the definitions in double precision (autograd for the gradients)."""
    s = prepare(case, seed)
    kind = s["kind"]
    f = torch.float64
    if kind in ("cache", "rope"):
        r0, R = s["start"], s["R"]
        theta = s["positions"].to(f)[:, :, None, None] * s["inv_freq"].to(f)
        turn = torch.polar(torch.ones_like(theta), theta)

        def rotated(x):
            part = x[..., r0:r0 + R]
            part = part.unflatten(-1, (R // 2, 2)) if s["interleaved"] else part.unflatten(-1, (2, R // 2)).transpose(-1, -2)
            part = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
            part = part.flatten(-2) if s["interleaved"] else part.transpose(-1, -2).flatten(-2)
            return torch.cat((x[..., :r0], part, x[..., r0 + R:]), -1)

        def normed(x, n, how, w, b):
            if how == "none":
                return x
            h = x[..., :n]
            if how == "layer":
                h = (h - h.mean(-1, keepdim=True)) / torch.sqrt(h.var(-1, unbiased=False, keepdim=True) + _EPS)
            else:
                h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + _EPS)
            h = h * w if b is None else h * w + b
            return torch.cat((h, x[..., n:]), -1)

    if kind == "cache":
        n = s["D"] - s["R"]
        q = rotated(s["q"].to(f))
        k = rotated(normed(s["k"].to(f), n, "rms", s["k_weight"].to(f), None)).flatten(0, 2)
        slots = s["slots"].flatten().long()
        cache = s["cache"].to(f)
        if s["cache_rope"] is None:
            cache.view(-1, s["D"]).index_copy_(0, slots, k)
            return [q, cache]
        rope = s["cache_rope"].to(f)
        cache.view(-1, n).index_copy_(0, slots, k[:, :n].contiguous())
        rope.view(-1, R).index_copy_(0, slots, k[:, n:].contiguous())
        return [q, cache, rope]
    if kind == "rope":
        names = [n for n in ("q", "k", "q_weight", "q_bias", "k_weight", "k_bias") if s[n] is not None]
        d = {n: s[n].detach().to(f).requires_grad_(True) for n in names}
        q = rotated(normed(d["q"], s["norm_dim"], s["q_norm"], d.get("q_weight"), d.get("q_bias")))
        k = rotated(normed(d["k"], s["norm_dim"], s["k_norm"], d.get("k_weight"), d.get("k_bias")))
        grads = torch.autograd.grad((q, k), [d[n] for n in names], (s["grad_q"].to(f), s["grad_k"].to(f)))
        return dict({"d_" + n: x for n, x in zip(names, grads)}, q=q.detach(), k=k.detach())
    if kind == "weights":
        B, S, H, D = s["q"].shape
        out = torch.zeros(s["indices"].shape, dtype=f, device=s["q"].device)
        for b in range(B):
            keys = s["kv"][b, :, 0].to(f)
            for t in range(S):
                idx = s["indices"][b, t, 0]
                idx = idx[idx >= 0].long()   # (a list's entries come before its padding)
                logits = s["q"][b, t].to(f) @ keys[idx].T / math.sqrt(D)
                out[b, t, 0, :idx.numel()] = torch.exp(logits - s["lse"][b, t].to(f)[:, None]).sum(0) / H
        return out
    if kind == "distill":
        rows, V = s["student"].shape
        losses, grads = torch.zeros(rows, dtype=f, device=s["teacher"].device), torch.zeros((rows, V), dtype=f, device=s["teacher"].device)
        for r in range(rows):
            row = s["student"][r].detach().to(f).requires_grad_(True)
            loss = _exact_row_loss(row, s["teacher"][r].to(f), None if s["indices"] is None else s["indices"][r].long(), s["over"], s["teacher_kind"], s["T"])
            losses[r] = loss.detach()
            grads[r] = torch.autograd.grad(loss, row, s["grad"][r].to(f))[0]
        return [losses, grads]
    query, key, weights = (s[n].detach().to(f) for n in ("query", "key", "weights"))
    B, S, H, _ = query.shape
    loss = torch.zeros((B, S), dtype=f, device=key.device)
    d_query, d_key, d_weights = torch.zeros_like(query), torch.zeros_like(key), torch.zeros_like(weights)
    for b in range(B):
        for t in range(S):
            idx = s["indices"][b, t, 0]
            there = idx >= 0
            idx = idx[there].long()
            values = s["values"][b, t, 0][there].to(f)
            p = s["teacher"][b, t, 0][there].to(f)
            p = p / p.sum()
            log_s = torch.log_softmax(values, 0)
            loss[b, t] = torch.special.xlogy(p, p).sum() - (p * log_s).sum()
            dv = s["grad"][b, t].to(f) * (log_s.exp() - p)
            rows = key[b, idx, 0]
            z = rows @ query[b, t].T
            d_weights[b, t] = dv @ z.clamp(min=0)
            dz = torch.where(z > 0, dv[:, None] * weights[b, t], torch.zeros_like(z))
            d_query[b, t] = dz.T @ rows
            d_key[b, :, 0].index_add_(0, idx, dz @ query[b, t])
    return [loss, d_query, d_key, d_weights]


def _exact_row_loss(student, teacher, columns, over, teacher_kind, T):
    z = student / T
    at = z if columns is None else z[columns]
    there = torch.isfinite(at.detach())
    t = teacher[there]
    p = torch.softmax(t / T, 0) if teacher_kind == "logits" else t / t.sum()
    norm = z[torch.isfinite(z.detach())] if over == "row" else at[there]
    return torch.special.xlogy(p, p).sum() - (p * (at[there] - torch.logsumexp(norm, 0))).sum()
