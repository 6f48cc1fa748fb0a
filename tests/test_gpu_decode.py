"""The one-kernel layer for a few tokens (decode.moe_layer, routed_layer)
against its formula in 64 bits.

Tolerance, elementwise and derived from the arithmetic: the products are
exact in fp32, a sum of n of them is off by at most n * 2^-23 of the sum of
their magnitudes; silu has a slope of at most 1.1; h = silu(gate) * up is
rounded once to bf16 (half a step, 2^-8 of the value) after fp32 arithmetic
(2^-20 covers expf and the divisions); y is rounded once to bf16.  Over all
elements two independent roundings of at most 2^-8, uniform within the step,
leave a relative error of at most sqrt(2/3) * 2^-8 < 2^-8 in the 2-norm."""
import pytest
import torch

from nvshmem_testing_b200 import _native as N
from nvshmem_testing_b200 import decode

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


def reference(x, ids, vals, w13, w2, first=0):
    """(y, bound) in 64 bits; an id counts once per row."""
    T, H = x.shape
    El, F, _ = w2.shape
    y = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(y)
    xd = x.double()
    for t in range(T):
        seen = set()
        for k, i in enumerate(ids[t].tolist()):
            e = i - first
            if not 0 <= e < El or i in seen:
                continue
            seen.add(i)
            w, d = w13[e].double(), w2[e].double()
            a, mag = xd[t] @ w, xd[t].abs() @ w.abs()
            da = mag * H * 2.0 ** -23
            g, u, dg, du = a[:F], a[F:], da[:F], da[F:]
            s = g * torch.sigmoid(g)
            h = s * u
            dh = 1.1 * dg * u.abs() + (s.abs() + 1.1 * dg) * du + h.abs() * (HALF + 2.0 ** -20)
            v = float(vals[t, k])
            y[t] += v * (h @ d)
            tol[t] += abs(v) * ((dh + (h.abs() + dh) * (F + 4) * 2.0 ** -23) @ d.abs())
    return y, tol + y.abs() * HALF + 1e-30


def check(y, x, ids, vals, w13, w2, first=0):
    ref, tol = reference(x, ids, vals, w13, w2, first)
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} beyond the bound, worst {float((err / tol).max()):.2f}x"
    if ref.numel() >= 1024 and float(ref.norm()) > 0:
        assert float(err.norm() / ref.norm()) <= HALF
    return ref


def make(T, H, El, K, F, seed, E=None, scale=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    E = E or El
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = (scale * torch.randn(El, H, 2 * F, generator=g, device="cuda")).to(torch.bfloat16)
    w2 = (scale * torch.randn(El, F, H, generator=g, device="cuda")).to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1).indices
    vals = torch.randn(T, K, generator=g, device="cuda").softmax(-1)
    return x, ids, vals, w13, w2


SIZES = [
    # T, H, E, K, F
    (1, 8, 1, 1, 8),
    (1, 64, 4, 1, 64),
    (1, 2048, 6, 6, 1408),
    (2, 72, 3, 3, 136),
    (3, 136, 5, 2, 72),
    (15, 520, 9, 4, 328),
    (16, 256, 8, 4, 128),
    (17, 264, 7, 3, 200),
    (31, 4096, 2, 2, 64),
    (33, 512, 16, 8, 384),
    (48, 64, 200, 5, 2048),
    (64, 1024, 32, 8, 256),
    (64, 256, 64, 16, 128),
    (64, 320, 1, 1, 1000),
    (56, 5000, 4, 4, 216),
    (40, 1032, 3, 3, 520),
]


@pytest.mark.parametrize("T,H,E,K,F", SIZES)
def test_known_routing(T, H, E, K, F):
    x, ids, vals, w13, w2 = make(T, H, E, K, F, T * 7 + H + F)
    y = decode.moe_layer(x, ids, vals, w13, w2)
    torch.cuda.synchronize()
    check(y, x, ids, vals, w13, w2)
    assert torch.equal(y, decode.moe_layer(x, ids, vals, w13, w2))  # sums in a fixed order


@pytest.mark.parametrize("T,H,E,K,F", [(5, 4096, 6, 2, 14344), (17, 4104, 7, 3, 12296), (33, 4096, 6, 2, 14344)])
def test_long_lists(T, H, E, K, F):
    """Enough weights that their last part is handed out in chunks (33 tokens:
    the same size without)."""
    x, ids, vals, w13, w2 = make(T, H, E, K, F, T, scale=0.02)
    y = decode.moe_layer(x, ids, vals, w13, w2)
    check(y, x, ids, vals, w13, w2)
    for _ in range(3):  # whoever takes a chunk, the sums are the same
        assert torch.equal(y, decode.moe_layer(x, ids, vals, w13, w2))


@pytest.mark.parametrize("T,H,E,K,F", [(18, 4360, 32, 3, 728), (9, 32768, 8, 2, 136), (32, 2056, 64, 4, 264),
                                       (33, 4352, 32, 3, 728), (1, 4096, 40, 32, 744)])
def test_long_lists_of_odd_rows(T, H, E, K, F):
    """Rows of w13 that are no multiple of 128 bytes: chunks from shorter lists
    on, many to a tile (33 tokens: fewer and larger ones)."""
    x, ids, vals, w13, w2 = make(T, H, E, K, F, T, scale=0.02)
    y = decode.moe_layer(x, ids, vals, w13, w2)
    check(y, x, ids, vals, w13, w2)
    for _ in range(3):
        assert torch.equal(y, decode.moe_layer(x, ids, vals, w13, w2))


@pytest.mark.parametrize("T,H,E,K,F", [(1, 64, 4, 2, 64), (3, 64, 4, 2, 64), (9, 72, 3, 3, 136), (40, 64, 2, 2, 64),
                                       (56, 1024, 4, 4, 72), (64, 1024, 32, 8, 64)])
def test_h_keeps_its_bits(T, H, E, K, F):
    """h = silu(gate) * up as two bf16 values: the second's rounding is half a
    step of what the first one's left, 2^-16 of h.  Beside it the terms of
    `reference`: fp32 sums of both products (twice as many terms in the
    second), y's rounding."""
    x, ids, vals, w13, w2 = make(T, H, E, K, F, T + F)
    y = decode.moe_layer(x, ids, vals, w13, w2).double()
    a = torch.einsum("th,ehf->etf", x.double(), w13.double())
    da = torch.einsum("th,ehf->etf", x.double().abs(), w13.double().abs()) * H * 2.0 ** -23
    g, u, dg, du = a[..., :F], a[..., F:], da[..., :F], da[..., F:]
    s = g * torch.sigmoid(g)
    h = s * u
    dh = 1.1 * dg * u.abs() + (s.abs() + 1.1 * dg) * du + h.abs() * (2.0 ** -16 + 2.0 ** -20)
    coef = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, ids, vals.double())
    ref = torch.einsum("te,eth->th", coef, h @ w2.double())
    tol = torch.einsum("te,eth->th", coef, (dh + (h.abs() + dh) * (2 * F + 4) * 2.0 ** -23) @ w2.double().abs())
    err = (y - ref).abs()
    tol = tol + (ref.abs() + tol) * HALF
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} beyond the bound, worst {float((err / tol).max()):.2f}x"


def test_h_beyond_the_types_range():
    """h above bf16's largest number goes on as infinity, not as NaN."""
    x = torch.full((3, 8), 1.0, dtype=torch.bfloat16, device="cuda")
    w13 = torch.zeros(1, 8, 32, dtype=torch.bfloat16, device="cuda")
    w13[0, :, 0], w13[0, :, 16] = 1e19, 1e19    # h = 6.4e39 at one feature
    w13[0, :, 1], w13[0, :, 17] = 0.25, 0.5     # and an ordinary one
    w2 = torch.zeros(1, 16, 8, dtype=torch.bfloat16, device="cuda")
    w2[0, 0, 3], w2[0, 1, 5] = -2.0, 1.0
    ids, vals = torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.ones(3, 1, device="cuda")
    y = decode.moe_layer(x, ids, vals, w13, w2)
    assert y[:, 3].tolist() == [-float("inf")] * 3


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("vals_dtype", [torch.float32, torch.bfloat16])
def test_types(ids_dtype, vals_dtype):
    x, ids, vals, w13, w2 = make(9, 256, 8, 3, 192, 5)
    ids, vals = ids.to(ids_dtype), vals.to(vals_dtype)
    check(decode.moe_layer(x, ids, vals, w13, w2), x, ids, vals, w13, w2)


def test_ids_elsewhere_repeated_and_negative():
    """A rank that holds experts [4, 9): other ids are skipped, a repeated id
    counts once with its first weight, a row without any id here is zero."""
    x, _, _, w13, w2 = make(6, 200, 5, 4, 104, 11)
    ids = torch.tensor([[4, 4, 5, 4], [0, 3, 9, 100], [8, 7, 6, 5], [-1, -5, 4, 12], [2 ** 31 - 1, 8, 8, 0],
                        [9, 9, 9, 9]], device="cuda")
    vals = torch.rand(6, 4, device="cuda") + 0.1
    for dt in (torch.int64, torch.int32):
        y = decode.moe_layer(x, ids.to(dt), vals, w13, w2, first_expert=4)
        check(y, x, ids, vals, w13, w2, first=4)
        assert not y[1].any() and not y[5].any()
    big = ids + (1 << 40)  # beyond 32 bits: matches nothing
    assert not decode.moe_layer(x, big, vals, w13, w2, first_expert=4).any()


def test_parts_of_the_experts_add_up():
    x, ids, vals, w13, w2 = make(12, 256, 8, 4, 128, 3)
    parts = sum(decode.moe_layer(x, ids, vals, w13[a:a + 2].contiguous(), w2[a:a + 2].contiguous(),
                                 first_expert=a).double() for a in range(0, 8, 2))
    ref, tol = reference(x, ids, vals, w13, w2)
    # four roundings of parts no larger than their magnitudes: the bound's own terms, once per part
    assert bool(((parts - ref).abs() <= 4 * tol + 4 * HALF * ref.abs() + 0.02 * tol.max()).all())


def test_no_expert_here_and_no_token():
    x, ids, vals, w13, w2 = make(5, 128, 4, 2, 64, 1)
    out = torch.full_like(x, 3.0)
    assert decode.moe_layer(x, ids + 4, vals, w13, w2, out=out) is out and not out.any()
    assert decode.moe_layer(x[:0], ids[:0], vals[:0], w13, w2).shape == (0, 128)


@pytest.mark.parametrize("T,H,F", [(1, 64, 72), (5, 7168, 256), (40, 1032, 520), (64, 4096, 728)])
def test_an_empty_rank(T, H, F):
    """No token has an expert here: every row is written, and zero."""
    x, ids, vals, w13, w2 = make(T, H, 3, 2, F, T)
    status = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    rw = torch.randn(H, 8, device="cuda").to(torch.bfloat16)
    for _ in range(3):
        out = torch.full_like(x, float("nan"))
        decode.moe_layer(x, ids, vals, w13, w2, first_expert=3, out=out, status=status)
        routed = decode.routed_layer(x, rw, 2, w13, w2, first_expert=8, status=status)[0]
        torch.cuda.synchronize()
        assert bool((out == 0).all()) and bool((routed == 0).all()) and int(status[0]) == 0


def test_a_token_is_touched_by_its_own_experts_only():
    """Non-finite tokens and experts stay with the rows that use them."""
    x, ids, vals, w13, w2 = make(8, 192, 4, 1, 96, 21)
    ids = torch.tensor([[0], [1], [2], [0], [1], [2], [0], [1]], device="cuda")
    clean = decode.moe_layer(x, ids, vals, w13, w2)
    x2, w13b, w2b = x.clone(), w13.clone(), w2.clone()
    x2[3] = float("nan")
    w13b[3] = float("nan")  # an expert that no token chose
    w2b[2, 5, 7] = float("inf")
    y = decode.moe_layer(x2, ids, vals, w13b, w2b)
    keep = [0, 1, 4, 6, 7]
    assert torch.equal(y[keep], clean[keep])
    assert bool(y[3].isnan().all())
    assert not bool(y[[2, 5]][:, 7].isfinite().any())
    assert bool(y[[2, 5]][:, :7].isfinite().all())


def test_strides_and_given_output():
    x, ids, vals, w13, w2 = make(7, 256, 6, 2, 128, 4)
    ref = decode.moe_layer(x, ids, vals, w13, w2)
    wide = torch.zeros(7, 512, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = x
    idt = torch.zeros(2, 7, dtype=torch.int64, device="cuda")
    idt.copy_(ids.t())
    rows = torch.full((9, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    y = decode.moe_layer(wide[:, ::2], idt.t(), vals.t().contiguous().t(), w13, w2, out=rows[1:8])
    assert torch.equal(y, ref)
    assert bool((rows[0] == 5).all()) and bool((rows[8] == 5).all())


def test_misaligned_and_misplaced_tensors_are_refused():
    x, ids, vals, w13, w2 = make(4, 128, 4, 2, 64, 1)
    flat = torch.zeros(4 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    odd = flat[1:1 + 4 * 128].view(4, 128)  # contiguous, 2 bytes off
    with pytest.raises(N.MoeEpError):
        decode.moe_layer(odd, ids, vals, w13, w2)
    with pytest.raises(N.MoeEpError):
        decode.moe_layer(x, ids, vals, w13, w2, out=odd)
    for bad in (dict(w13=w13.cpu()), dict(w2=w2.transpose(1, 2)), dict(top_vals=vals.cpu()), dict(first_expert=-1),
                dict(first_expert=1 << 31), dict(top_vals=vals.half()), dict(top_idxs=ids.float()),
                dict(top_idxs=ids[:3]), dict(out=x[:, :64])):
        with pytest.raises((ValueError, TypeError)):
            decode.moe_layer(**{**dict(x=x, top_idxs=ids, top_vals=vals, w13=w13, w2=w2), **bad})
    with pytest.raises(ValueError):
        decode.moe_layer(x.repeat(20, 1), ids.repeat(20, 1), vals.repeat(20, 1), w13, w2)  # 80 tokens
    rw = torch.zeros(128, 8, dtype=torch.bfloat16, device="cuda")
    for k, r in ((0, rw), (9, rw), (2, rw[:, :6]), (2, rw[:64]), (2, rw.cpu())):
        with pytest.raises(ValueError):
            decode.routed_layer(x, r, k, w13, w2)


def test_captured_and_replayed_beside_eager_calls():
    x, ids, vals, w13, w2 = make(4, 256, 8, 2, 128, 8)
    static, sids = x.clone(), ids.clone()
    decode.moe_layer(static, sids, vals, w13, w2)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decode.moe_layer(static, sids, vals, w13, w2))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        x2, ids2, _, _, _ = make(4, 256, 8, 2, 128, 100 + i)
        static.copy_(x2)
        sids.copy_(ids2)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = decode.moe_layer(x2, ids2, vals, w13, w2)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)


def test_several_streams_at_once():
    data = [make(3 + 5 * i, 512, 16, 4, 256, 40 + i) for i in range(4)]
    want = [decode.moe_layer(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for d, s in zip(data, streams):
            with torch.cuda.stream(s):
                got.append(decode.moe_layer(*d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


ROUTED = [
    # T, H, E, K, F
    (1, 64, 4, 1, 64),
    (1, 2048, 64, 6, 128),
    (2, 7168, 256, 8, 64),
    (5, 136, 12, 3, 72),
    (13, 520, 104, 5, 64),
    (40, 256, 1024, 4, 16),
    (64, 1000, 128, 8, 64),
    (64, 64, 700, 16, 8),
    (32, 128, 32, 32, 64),
]


@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("T,H,E,K,F", ROUTED)
def test_router(T, H, E, K, F, renormalize):
    x, _, _, w13, w2 = make(T, H, E, K, F, T + H + E)
    g = torch.Generator(device="cuda").manual_seed(E)
    rw = (torch.randn(H, E, generator=g, device="cuda") / H ** 0.5).to(torch.bfloat16)
    dt = torch.int32 if renormalize else torch.int64
    y, vals, ids = decode.routed_layer(x, rw, K, w13, w2, renormalize=renormalize, ids_dtype=dt)
    torch.cuda.synchronize()
    assert ids.dtype == dt and vals.dtype == torch.float32 and ids.shape == vals.shape == (T, K)
    logits = x.double() @ rw.double()
    slack = (x.double().abs() @ rw.double().abs()) * (H + 4) * 2.0 ** -24  # fp32 sums of H products
    chosen = torch.gather(logits, 1, ids.long())
    near = 2 * slack.amax(dim=1, keepdim=True)
    # descending within the slack, distinct, and nothing left out is larger
    assert bool((chosen[:, 1:] <= chosen[:, :-1] + near).all())
    assert all(len(set(r)) == K for r in ids.tolist())
    rest = logits.scatter(1, ids.long(), float("-inf")).amax(dim=1, keepdim=True)
    assert bool((rest <= chosen[:, -1:] + near).all())
    prob = torch.softmax(logits, -1).gather(1, ids.long())
    if renormalize:
        prob = prob / prob.sum(-1, keepdim=True)
    # logits off by `slack`, then expf, sum (E terms) and division in fp32
    rel = torch.expm1(2 * near) + (E + K + 16) * 2.0 ** -23
    assert bool(((vals.double() - prob).abs() <= prob * rel).all())
    check(y, x, ids, vals, w13, w2)
    # the same result as the layer with that routing given
    assert torch.equal(y, decode.moe_layer(x, ids, vals, w13, w2))


def test_router_ties_and_part_of_the_experts():
    T, H, E, K, F = 6, 128, 32, 4, 64
    x, _, _, w13, w2 = make(T, H, 8, K, F, 77)
    rw = torch.zeros(H, E, dtype=torch.bfloat16, device="cuda")
    _, vals, ids = decode.routed_layer(x, rw, K, w13, w2, first_expert=0)
    assert ids.tolist() == [list(range(K))] * T  # equal logits: lowest ids
    assert bool((vals == 1.0 / E).all())
    rw[:, 20:] = (0.1 * torch.randn(H, 12, device="cuda")).to(torch.bfloat16)
    y, vals, ids = decode.routed_layer(x, rw, K, w13, w2, first_expert=20)
    check(y, x, ids, vals, w13, w2, first=20)


def test_router_with_non_finite_tokens():
    """A NaN token keeps to its own row and its ids stay valid."""
    T, H, E, K, F = 5, 256, 16, 3, 64
    x, _, _, w13, w2 = make(T, H, E, K, F, 2)
    rw = (0.1 * torch.randn(H, E, device="cuda")).to(torch.bfloat16)
    ref, vals0, ids0 = decode.routed_layer(x, rw, K, w13, w2)
    x2 = x.clone()
    x2[2, 9] = float("nan")
    y, vals, ids = decode.routed_layer(x2, rw, K, w13, w2)
    keep = [0, 1, 3, 4]
    assert torch.equal(ids[keep], ids0[keep]) and torch.equal(vals[keep], vals0[keep])
    assert torch.equal(y[keep], ref[keep])
    assert bool(((ids >= 0) & (ids < E)).all()) and bool(y[2].isnan().all())


@pytest.mark.parametrize("E", [16, 200])  # both ways to find the largest
@pytest.mark.parametrize("T", [1, 7])
@pytest.mark.parametrize("renormalize", [False, True])
def test_router_with_infinite_logits(T, E, renormalize):
    """Logits of minus infinity have weight 0 and come last, by id; plus
    infinity comes first and leaves no softmax (NaN weights, valid ids), as
    the softmax's definition has it; a token's row concerns itself only."""
    H, K, F = 256, 6, 64
    x, _, _, w13, w2 = make(T, H, 4, 1, F, E)
    x = x.abs() + 1
    rw = (0.1 * torch.randn(H, E, generator=torch.Generator(device="cuda").manual_seed(E), device="cuda")).to(
        torch.bfloat16)
    finite = [3, 5, 11, E - 2]
    low = torch.full_like(rw, float("-inf"))
    low[:, finite] = rw[:, finite]
    y, vals, ids = decode.routed_layer(x, low, K, w13, w2, renormalize=renormalize)
    logits = x.double() @ low.double()
    prob = torch.softmax(logits, -1)  # of the four finite ones
    for t in range(T):
        assert sorted(ids[t, :4].tolist()) == sorted(finite)
        assert ids[t, 4:].tolist() == [0, 1]  # of the rest the lowest ids
    # fp32 logits (each off by `slack` at most), expf, the sum and the division
    slack = (x.double().abs() @ rw.double().abs()).amax() * (H + 4) * 2.0 ** -24
    rel = torch.expm1(4 * slack) + (E + K + 16) * 2.0 ** -23
    assert bool(((vals.double() - prob.gather(1, ids)).abs() <= prob.gather(1, ids) * rel).all())
    check(y, x, ids, vals, w13, w2)
    high = rw.clone()
    high[:, E // 2] = float("inf")
    y, vals, ids = decode.routed_layer(x, high, K, w13, w2, renormalize=renormalize)
    assert bool((ids[:, 0] == E // 2).all()) and bool(vals.isnan().all())
    assert bool(((ids >= 0) & (ids < E)).all()) and all(len(set(r)) == K for r in ids.tolist())
    if T > 1:  # one token's infinity
        x2 = x.clone()
        x2[2, 9] = float("inf")
        ref = decode.routed_layer(x, rw, K, w13, w2, renormalize=renormalize)
        got = decode.routed_layer(x2, rw, K, w13, w2, renormalize=renormalize)
        keep = [t for t in range(T) if t != 2]
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, ref))
        assert bool(((got[2] >= 0) & (got[2] < E)).all()) and bool(got[1][2].isnan().all())


def test_status_word_stays_clear():
    x, ids, vals, w13, w2 = make(4, 128, 4, 2, 64, 6)
    status = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    decode.moe_layer(x, ids, vals, w13, w2, status=status)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
