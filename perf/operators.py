"""The package's decode and 8-bit operators as measurable cases.

Four operators of a mixture-of-experts model's serving path:

* ``routed``  the whole layer for a few tokens from activations: router,
  gated expert MLP, weighted sum over the chosen experts;
* ``decode``  the same layer for routing that is already known, on a rank that
  holds experts [first, first + El) of E;
* ``product`` 8-bit integer product with a scale per row and per channel, one
  weight matrix per expert, rows in expert order (``linear`` is the dense form
  from bf16 rows, which are quantised on the way);
* ``layer8``  the gated expert layer in 8 bits, from bf16 rows to bf16 rows.

``run`` takes the plain torch form of each, or the package's own call where
``own`` is true.
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of an interactive session; a layer of 64 small experts: latency counts.
        dict(name="routed_t1_e64", op="routed", T=1, H=2048, E=64, K=6, F=1408),
        # One token, 256 experts of 88 MB each: a stream of weights.
        dict(name="routed_t1_e256", op="routed", T=1, H=7168, E=256, K=8, F=2048),
        # A decode batch over the 64 small experts: nearly all of them are active.
        dict(name="routed_t32_e64", op="routed", T=32, H=2048, E=64, K=6, F=1408),
        # An odd batch over eight wide experts, routing known.
        dict(name="decode_t7_e8", op="decode", T=7, H=4096, E=8, El=8, first=0, K=2, F=14336),
        # The largest batch, on a rank that holds 64 of 256 experts.
        dict(name="decode_t64_shard", op="decode", T=64, H=7168, E=256, El=64, first=64, K=8, F=2048),
        # 8-bit product of a rank of eight: 32 experts with about 1000 rows each.
        dict(name="product_large", op="product", rows=32768, K=7168, N=4096, E=32, alpha=0.0),
        # The same with skewed experts: some crowded, some nearly empty.
        dict(name="product_skewed", op="product", rows=6145, K=2048, N=2816, E=64, alpha=1.2),
        # A few rows in each of eight experts: the weights' bytes count.
        dict(name="product_few_rows", op="product", rows=21, K=4096, N=14336, E=8, alpha=0.0),
        # A dense projection for one token, from bf16.
        dict(name="linear_one_row", op="linear", rows=1, K=7168, N=4096),
        # A dense projection for a prefill, from bf16.
        dict(name="linear_prefill", op="linear", rows=4096, K=4096, N=14336),
        # The gated layer in 8 bits, a prefill over eight wide experts.
        dict(name="layer8_prefill_e8", op="layer8", T=4096, H=4096, E=8, El=8, first=0, K=2, F=14336),
        # The gated layer in 8 bits for a decode batch on a rank with 32 of 256 experts.
        dict(name="layer8_t257_shard", op="layer8", T=257, H=7168, E=256, El=32, first=96, K=8, F=2048),
    ]


def _log(rng, lo, hi, step=1):
    """A whole number of [lo, hi], a multiple of step, spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("routed", "decode", "product", "linear", "layer8"))
    if op in ("routed", "decode"):
        E = rng.choice((4, 8, 16, 24, 48, 64, 104, 128, 192, 256))
        H, F = _log(rng, 256, 7168, 8), _log(rng, 128, 14336, 8)
        while E * H * F > 54 * 7168 * 2048:
            E, F = (E // 2 if E > 8 else E), F // 16 * 8 if E <= 8 else F
        c = dict(op=op, T=_log(rng, 1, 64), H=H, E=E, K=rng.randint(1, min(8, E)), F=F)
        if op == "decode":
            El = rng.choice((E, E, max(1, E // 2), max(1, E // 4)))
            c.update(El=El, first=rng.randint(0, E - El))
        return c
    if op == "product":
        E = rng.choice((1, 2, 8, 24, 32, 64))
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, K=_log(rng, 256, 7168, 16), N=_log(rng, 256, 7168, 8), E=E,
                    alpha=rng.choice((0.0, 1.2)) if rows <= 8192 else 0.0)
    if op == "linear":
        return dict(op=op, rows=_log(rng, 1, 4096), K=_log(rng, 256, 7168, 16), N=_log(rng, 256, 14336, 8))
    E = rng.choice((4, 8, 32, 64))
    El = rng.choice((E, max(1, E // 2)))
    return dict(op=op, T=_log(rng, 1, 2048), H=_log(rng, 256, 4096, 16), E=E, El=El, first=rng.randint(0, E - El),
                K=rng.randint(1, min(6, E)), F=_log(rng, 256, 4096, 16))


# ------------------------------------------------------------------ inputs
def _weights(g, shape):
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, 0.02, generator=g)


def _weights8(g, E, N, K):
    """8-bit weights as a quantiser with a scale per channel leaves them."""
    q = torch.empty((E, N, K), dtype=torch.bfloat16, device=DEV).normal_(0.0, 32.0, generator=g)
    q = q.round_().clamp_(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand((E, N), generator=g, device=DEV)) * (0.02 / 32)
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    c, s = case, dict(op=case["op"])
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    if c["op"] == "product":
        p = torch.arange(1, c["E"] + 1, device=DEV, dtype=torch.float64).pow(-c["alpha"])
        p = p[torch.randperm(c["E"], generator=g, device=DEV)]
        owner = torch.multinomial(p, c["rows"], replacement=True, generator=g)
        s["counts"] = torch.bincount(owner, minlength=c["E"]).to(torch.int32)
        s["wq"], s["ws"] = _weights8(g, c["E"], c["N"], c["K"])
        s["xq"] = (randn(c["rows"], c["K"]) * 32).round().clamp(-127, 127).to(torch.int8)
        s["xs"] = (0.5 + torch.rand(c["rows"], generator=g, device=DEV)) / 32
        return s
    if c["op"] == "linear":
        s["x"] = randn(c["rows"], c["K"]).to(torch.bfloat16)
        s["wq"], s["ws"] = _weights8(g, 1, c["N"], c["K"])
        return s
    T, H, E, K, F = c["T"], c["H"], c["E"], c["K"], c["F"]
    s["x"] = randn(T, H).to(torch.bfloat16)
    s["K"] = K
    if c["op"] == "routed":
        s["router_w"] = _weights(g, (H, E))
    else:
        s["first"] = c["first"]
        s["ids"] = torch.rand((T, E), generator=g, device=DEV).topk(K, dim=-1).indices
        s["vals"] = randn(T, K).softmax(dim=-1)
    El = c.get("El", E)
    if c["op"] == "layer8":
        s["w13q"], s["w13s"] = _weights8(g, El, 2 * F, H)
        s["w2q"], s["w2s"] = _weights8(g, El, H, F)
    else:
        s["w13"], s["w2"] = _weights(g, (El, H, 2 * F)), _weights(g, (El, F, H))
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_experts(x, ids, vals, w13, w2, first):
    """Every token through every expert that any token chose, then the
    chosen ones' weighted sum."""
    F = w2.shape[1]
    local = ids - first
    active = torch.unique(local[(local >= 0) & (local < w13.shape[0])])
    if active.numel() == 0:
        return torch.zeros_like(x)
    a = torch.matmul(x.float(), w13[active].float())                                  # [A, T, 2F]
    gate, up = a[..., :F], a[..., F:]
    out = torch.matmul(gate / (1 + torch.exp(-gate)) * up, w2[active].float())        # [A, T, H]
    coef = (vals * (local == active[:, None, None])).sum(-1)                          # [A, T]
    return (coef[..., None] * out).sum(0).to(x.dtype)


def _plain_quantize(x):
    """[rows, K] -> whole numbers in [-127, 127] and a scale per row; the
    quotient is taken in 64 bits, where it cannot be rounded onto a border."""
    scale = x.float().abs().amax(dim=-1) / 127
    q = (x.double() / scale.double()[:, None]).nan_to_num_(0.0).round_().clamp_(-127, 127)
    return q.float(), scale


def _plain_bucketed(rows, scale, expert, E, wq, ws):
    """Products of rows (sorted by expert) with their experts' matrices, as
    one batched product over buckets padded to the largest."""
    counts = torch.bincount(expert, minlength=E)
    pos = torch.arange(rows.shape[0], device=rows.device) - (counts.cumsum(0) - counts)[expert]
    buf = torch.zeros((E, max(int(counts.max()), 1), rows.shape[1]), device=rows.device)
    buf[expert, pos] = rows
    out = torch.matmul(buf, wq.float().transpose(1, 2))[expert, pos]
    return out * scale[:, None] * ws[expert]


def _plain_layer8(s):
    x, ids, vals, K = s["x"], s["ids"], s["vals"], s["K"]
    El, F = s["w2q"].shape[0], s["w2q"].shape[2]
    local = (ids - s["first"]).reshape(-1)
    local = torch.where((local >= 0) & (local < El), local, El)
    order = torch.argsort(local, stable=True)
    order = order[: int((local < El).sum())]
    if order.numel() == 0:
        return torch.zeros_like(x)
    expert, token = local[order], order // K
    q, scale = _plain_quantize(x)
    a = _plain_bucketed(q[token], scale[token], expert, El, s["w13q"], s["w13s"])
    gate, up = a[:, :F], a[:, F:]
    q, scale = _plain_quantize(gate / (1 + torch.exp(-gate)) * up)
    out = _plain_bucketed(q, scale, expert, El, s["w2q"], s["w2s"])
    y = torch.zeros((x.shape[0] * K, x.shape[1]), device=x.device)
    y[order] = out * vals.reshape(-1)[order][:, None]
    return y.view(x.shape[0], K, -1).sum(1).to(x.dtype)


def _run_plain(s):
    if s["op"] == "routed":
        # Logits in 64 bits: which expert is chosen hangs on the difference of near ones.
        prob = torch.softmax(s["x"].double() @ s["router_w"].double(), dim=-1)
        vals, ids = torch.sort(prob, dim=-1, descending=True, stable=True)
        vals, ids = vals[:, : s["K"]].float().contiguous(), ids[:, : s["K"]].contiguous()
        return {"y": _plain_experts(s["x"], ids, vals, s["w13"], s["w2"], 0), "vals": vals, "ids": ids}
    if s["op"] == "decode":
        return _plain_experts(s["x"], s["ids"], s["vals"], s["w13"], s["w2"], s["first"])
    if s["op"] == "product":
        E = s["wq"].shape[0]
        expert = torch.repeat_interleave(torch.arange(E, device=DEV), s["counts"].long())
        return _plain_bucketed(s["xq"].float(), s["xs"], expert, E, s["wq"], s["ws"]).to(torch.bfloat16)
    if s["op"] == "linear":
        q, scale = _plain_quantize(s["x"])
        return (q @ s["wq"][0].float().t() * scale[:, None] * s["ws"][0]).to(torch.bfloat16)
    return _plain_layer8(s)


# ------------------------------------------------------------------ the package's calls
def _run_own(s):
    from nvshmem_testing_b200 import decode, w8a8
    if s["op"] == "routed":
        y, vals, ids = decode.routed_layer(s["x"], s["router_w"], s["K"], s["w13"], s["w2"])
        return {"y": y, "vals": vals, "ids": ids}
    if s["op"] == "decode":
        return decode.moe_layer(s["x"], s["ids"], s["vals"], s["w13"], s["w2"], first_expert=s["first"])
    if s["op"] == "product":
        return w8a8.grouped_gemm(s["xq"], s["xs"], w8a8.QuantWeights(s["wq"], s["ws"]), s["counts"])
    if s["op"] == "linear":
        return w8a8.linear(s["x"], w8a8.QuantWeights(s["wq"], s["ws"]))
    return w8a8.moe_layer(s["x"], s["ids"], s["vals"], w8a8.QuantWeights(s["w13q"], s["w13s"]),
                          w8a8.QuantWeights(s["w2q"], s["w2s"]), first_expert=s["first"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without
def _active(El, E, K, T):
    """Experts of El that some of T tokens choose (K of E each), on average."""
    return El * (1.0 - (1.0 - K / E) ** T)


def work(case):
    c = case
    if c["op"] in ("product", "linear"):
        E = c.get("E", 1)
        used = min(E, c["rows"]) if not c.get("alpha") else E * 0.9
        w = used * c["N"] * c["K"]
        return {"bytes": w + c["rows"] * (c["K"] * (2 if c["op"] == "linear" else 1) + 2 * c["N"]),
                "flops": 2 * c["rows"] * c["N"] * c["K"]}
    T, H, E, K, F = c["T"], c["H"], c["E"], c["K"], c["F"]
    El = c.get("El", E)
    width = 1 if c["op"] == "layer8" else 2
    pairs = T * K * El / E
    return {"bytes": _active(El, E, K, T) * 3 * H * F * width + 4 * T * H + (2 * H * E if c["op"] == "routed" else 0),
            "flops": pairs * 6 * H * F}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_silu_mul(a):
    g, u = a.chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u


def _exact_pairs(ids, first, El):
    """Per local expert: the (token, k) pairs that chose it."""
    flat = ids.cpu()
    for e in range(El):
        t, k = (flat == first + e).nonzero(as_tuple=True)
        if t.numel():
            yield e, t.to(DEV), k.to(DEV)


def _exact_quantize(x):
    """The whole numbers and their row's scale (held in 32 bits by definition)."""
    top = x.abs().max(dim=1, keepdim=True).values
    scale = (top.float() / 127).double()
    return torch.clamp(torch.round(torch.where(top > 0, x / scale, 0.0)), -127, 127), scale


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "product":
        out = torch.empty((s["xq"].shape[0], s["wq"].shape[1]), dtype=torch.float64, device=DEV)
        at = 0
        for e, n in enumerate(s["counts"].tolist()):
            out[at:at + n] = (s["xq"][at:at + n].double() * s["xs"][at:at + n].double()[:, None]) @ \
                (s["wq"][e].double() * s["ws"][e].double()[:, None]).t()
            at += n
        return out
    x = s["x"].double()
    if op == "linear":
        q, scale = _exact_quantize(x)
        return (q * scale) @ (s["wq"][0].double() * s["ws"][0].double()[:, None]).t()
    got = {}
    if op == "routed":
        logits = torch.einsum("th,he->te", x, s["router_w"].double())
        prob = torch.exp(logits - torch.logsumexp(logits, dim=1, keepdim=True))
        rank = torch.argsort(-logits, dim=1, stable=True)[:, : s["K"]]
        got = {"ids": rank, "vals": torch.gather(prob, 1, rank)}
        ids, vals, first = rank, got["vals"], 0
    else:
        ids, vals, first = s["ids"], s["vals"].double(), s["first"]
    y = torch.zeros_like(x)
    if op == "layer8":
        for e, t, k in _exact_pairs(ids, first, s["w2q"].shape[0]):
            q, scale = _exact_quantize(x[t])
            a = (q * scale) @ (s["w13q"][e].double() * s["w13s"][e].double()[:, None]).t()
            q, scale = _exact_quantize(_exact_silu_mul(a))
            o = (q * scale) @ (s["w2q"][e].double() * s["w2s"][e].double()[:, None]).t()
            y.index_add_(0, t, o * vals[t, k][:, None])
        return y
    for e, t, k in _exact_pairs(ids, first, s["w2"].shape[0]):
        h = _exact_silu_mul(x[t] @ s["w13"][e].double())
        y.index_add_(0, t, (h @ s["w2"][e].double()) * vals[t, k][:, None])
    return {"y": y, **got} if op == "routed" else y
