"""8-bit quantisation, products and the gated layer (w8a8) against their
definitions in 64 bits.

Tolerances, derived from the arithmetic: the quantisation is exact (equality);
a product's integer sum is exact, its conversion and two scale products round
by 2^-24 each (2^-22 in all), the bf16 output by half a step, 2^-8; silu has a
slope of at most 1.1 and its fp32 evaluation is covered by 2^-20."""
import pytest
import torch

from nvshmem_testing_b200 import _native as N
from nvshmem_testing_b200 import decode, utils, w8a8

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
RECIP = float(torch.tensor(1.0) / torch.tensor(127.0))  # 1/127 in fp32


def quant_ref(x):
    """(q, scale) by definition: the scale in fp32, the quotient in 64 bits
    (24-bit operands: no quotient is nearer to a tie than 2^-48 without being
    one)."""
    top = x.float().abs().amax(1)
    scale = top * RECIP
    q = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0).round().clamp(-127, 127)
    bad = ~torch.isfinite(x.float()).all(1)
    q[bad], scale[bad] = 0, float("nan")
    return q.to(torch.int8), scale


def check_quant(x, got, perm=None):
    q, s = quant_ref(x if perm is None else x[perm.long()])
    assert torch.equal(got[0], q)
    assert torch.equal(got[1].view(torch.int32)[~s.isnan()], s.view(torch.int32)[~s.isnan()])
    assert bool((got[1].isnan() == s.isnan()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 8), (3, 16), (5, 264), (7, 1408), (33, 2048), (9, 7168), (300, 4096),
                                    (2, 14336), (3, 40008), (5000, 72)])
def test_quantize_rows(rows, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + K)
    x = torch.randn(rows, K, generator=g, device="cuda").to(dtype)
    check_quant(x, w8a8.quantize_rows(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_ties_and_extremes(dtype):
    K = 512
    base = torch.arange(-256, 256, device="cuda").float() / 2  # every half step of a row with maximum 127
    rows = [base.clamp(-127, 127), base.clamp(-127, 127) * 2.0 ** -120, base * 2.0 ** 100,
            torch.zeros(K, device="cuda"), torch.full((K,), -3.0, device="cuda"),
            base.clamp(-127, 127) * 1.0078125, torch.linspace(-1, 1, K, device="cuda"),
            base.clamp(-127, 127) * 2.0 ** -133]
    x = torch.stack(rows).to(dtype)
    for scale in (1.0, 3.0, 0.7, 127.0 / 3):
        y = (x.float() * scale).to(dtype)
        check_quant(y, w8a8.quantize_rows(y))
    big = torch.finfo(dtype).max
    y = x.clone()
    y[0, 3], y[1, 0], y[2, 7], y[3, 1] = float("inf"), float("nan"), -float("inf"), big
    check_quant(y, w8a8.quantize_rows(y))


def test_quantize_gathers_and_leaves_the_rest():
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(50, 256, generator=g, device="cuda").to(torch.bfloat16)
    perm = torch.randint(0, 50, (333,), generator=g, device="cuda", dtype=torch.int32)
    check_quant(x, w8a8.quantize_rows(x, perm), perm)
    q = torch.full((333, 256), 77, dtype=torch.int8, device="cuda")
    s = torch.full((333,), 5.0, device="cuda")
    live = torch.tensor([101], dtype=torch.int32, device="cuda")
    far = perm.clone()
    far[101:] = 1 << 30  # behind the last live row: not even read from
    N.check(N.lib().moe_quant_rows(x.data_ptr(), 0, 333, 256, far.data_ptr(), live.data_ptr(), q.data_ptr(),
                                   s.data_ptr(), None), "moe_quant_rows")
    torch.cuda.synchronize()
    check_quant(x, (q[:101], s[:101]), perm[:101])
    assert bool((q[101:] == 77).all()) and bool((s[101:] == 5).all())


def test_quantize_weights_per_channel():
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(3, 48, 24, generator=g, device="cuda").to(torch.bfloat16)
    got = w8a8.quantize_weights(w)
    assert got.q.shape == (3, 24, 48) and got.scale.shape == (3, 24)
    for e in range(3):
        check_quant(w[e].t(), (got.q[e], got.scale[e]))


def make(rows, K, Nn, E, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xq = torch.randint(-127, 128, (rows, K), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(rows, generator=g, device="cuda") + 0.1
    wq = torch.randint(-127, 128, (E, Nn, K), generator=g, device="cuda", dtype=torch.int8)
    ws = (torch.rand(E, Nn, generator=g, device="cuda") + 0.1) / 127 / K ** 0.5
    return xq, xs / 127, wq, ws


def product_ref(xq, xs, wq, ws, counts):
    out = torch.zeros(sum(counts), wq.shape[1], dtype=torch.float64, device="cuda")
    at = 0
    for e, n in enumerate(counts):  # sums below 2^31: exact in 64 bits
        out[at:at + n] = (xq[at:at + n].double() @ wq[e].double().t()) * xs[at:at + n].double()[:, None] * ws[e].double()
        at += n
    return out


def glu_ref(a):
    """silu(gate) * up and how far fp32 arithmetic may be off."""
    g, u = a.chunk(2, 1)
    s = g * torch.sigmoid(g)
    d = 2.0 ** -22
    return s * u, (1.1 * g.abs() * u.abs() + s.abs() * u.abs()) * d + (s * u).abs() * 2.0 ** -20


PRODUCTS = [
    # K, N, counts
    (16, 8, [1]),
    (48, 24, [3, 0, 2]),
    (128, 256, [32]),
    (144, 264, [33, 1, 0, 31]),
    (400, 1000, [255, 256, 257]),
    (1408, 512, [5] * 40),
    (2048, 2816, [600, 0, 7, 1]),
    (7168, 320, [1]),
    (7168, 4096, [1, 2]),
    (7168, 512, [17]),
    (528, 72, [3]),
    (1040, 328, [2, 0, 4, 1, 5, 0, 4]),
    (6128, 256, [4, 0, 0, 12]),
    (6160, 256, [16]),
    (2048, 136, [9, 0, 14, 9]),
    (3088, 136, [5, 0, 14, 13] + [0] * 12),
    (1040, 4096, [1, 4, 3, 2, 0, 7]),
    (256, 4096, [1500, 2000, 1300]),   # whole tiles
    (512, 1536, [4090, 3841]),
]


@pytest.mark.parametrize("K,Nn,counts", PRODUCTS)
@pytest.mark.parametrize("swiglu", [False, True])
def test_products(K, Nn, counts, swiglu):
    rows = sum(counts)
    if swiglu:
        Nn = Nn // 16 * 16 if Nn >= 16 else 16
    xq, xs, wq, ws = make(rows, K, Nn, len(counts), rows + K + Nn)
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    w = w8a8.QuantWeights(wq, ws)
    ref = product_ref(xq, xs, wq, ws, counts)
    slack = ref.abs() * 2.0 ** -22
    if swiglu:
        ref, slack = glu_ref(ref)
    for dt, half in ((torch.float32, 2.0 ** -24), (torch.bfloat16, HALF)):
        out = w8a8.grouped_gemm(xq, xs, w, cd, swiglu=swiglu, out_dtype=dt)
        torch.cuda.synchronize()
        assert out.dtype == dt and out.shape == ref.shape
        err = (out.double() - ref).abs()
        tol = slack + (ref.abs() + slack) * half + 1e-37
        assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()}, worst {float((err / tol).max()):.2f}x"
        assert torch.equal(out, w8a8.grouped_gemm(xq, xs, w, cd, swiglu=swiglu, out_dtype=dt))


@pytest.mark.parametrize("rows,K", [(1, 16), (40, 16), (40, 8192), (9000, 16)])
def test_swiglu_of_far_gates(rows, K):
    """silu's values are far below 1 at gates of -80 to -88, not zero: a large
    up value brings them back."""
    gates = torch.arange(80, 88.7, 0.1, device="cuda")
    Nn = 2 * ((gates.numel() + 7) // 8 * 8)
    ws = torch.full((1, Nn), 1e30, device="cuda")
    ws[0, :Nn // 2] = -1.0
    ws[0, :gates.numel()] = -gates
    wq = torch.zeros(1, Nn, K, dtype=torch.int8, device="cuda")
    wq[..., 0] = 1
    xq = torch.zeros(rows, K, dtype=torch.int8, device="cuda")
    xq[:, 0] = 1
    out = w8a8.grouped_gemm(xq, torch.ones(rows, device="cuda"), w8a8.QuantWeights(wq, ws), swiglu=True,
                            out_dtype=torch.float32)
    a = ws[0].double()
    ref = a[:Nn // 2] * torch.sigmoid(a[:Nn // 2]) * a[Nn // 2:]
    assert bool(((out.double() - ref).abs() <= ref.abs() * 2.0 ** -20).all())


def test_many_experts_mostly_empty():
    counts = [0] * 1024
    for e in (0, 5, 511, 512, 1000, 1023):
        counts[e] = e % 7 + 1
    rows = sum(counts)
    xq, xs, wq, ws = make(rows, 32, 16, 1024, 3)
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = w8a8.grouped_gemm(xq, xs, w8a8.QuantWeights(wq, ws), cd, out_dtype=torch.float32)
    ref = product_ref(xq, xs, wq, ws, counts)
    assert bool(((out.double() - ref).abs() <= ref.abs() * 2.0 ** -21).all())


@pytest.mark.parametrize("Nn", [64, 4096])
def test_rows_behind_the_last_are_left(Nn):
    counts = [20, 3]
    xq, xs, wq, ws = make(700, 256, Nn, 2, 9)
    cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for glu in (False, True):
        out = torch.full((700, Nn // 2 if glu else Nn), 9.0, dtype=torch.bfloat16, device="cuda")
        assert w8a8.grouped_gemm(xq, xs, w8a8.QuantWeights(wq, ws), cd, swiglu=glu, out=out) is out
        ref = product_ref(xq, xs, wq, ws, counts)
        if glu:
            ref = glu_ref(ref)[0]
        assert bool((out[23:] == 9).all())
        assert bool(((out[:23].double() - ref).abs() <= ref.abs() * 1.01 * HALF + 1e-4 * ref.abs().max()).all())
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.full((700, Nn), 9.0, dtype=torch.bfloat16, device="cuda")
    w8a8.grouped_gemm(xq, xs, w8a8.QuantWeights(wq, ws), none, out=out)
    assert bool((out == 9).all())
    # counts past the last row are cut, negative ones count as none
    over = torch.tensor([-5, 100000], dtype=torch.int32, device="cuda")
    got = w8a8.grouped_gemm(xq, xs, w8a8.QuantWeights(wq, ws), over, out_dtype=torch.float32)
    ref = product_ref(xq, xs, wq, ws, [0, 700])
    assert bool(((got.double() - ref).abs() <= ref.abs() * 2.0 ** -21).all())


def test_largest_sums():
    """Every product at its extreme over the longest K: no sum wraps."""
    K = 131056
    xq = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    xq[1] = 127
    wq = torch.full((1, 8, K), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda"), torch.ones(1, 8, device="cuda")
    out = w8a8.grouped_gemm(xq, one[0], w8a8.QuantWeights(wq, one[1]), out_dtype=torch.float32)
    assert out[0].tolist() == [float(16384 * K)] * 8
    assert bool(((out[1].double() + 16256.0 * K).abs() <= 16256.0 * K * 2.0 ** -24).all())


def test_non_finite_rows_stay_apart():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(40, 512, generator=g, device="cuda").to(torch.bfloat16)
    w = w8a8.quantize_weights(torch.randn(1, 512, 256, generator=g, device="cuda").to(torch.bfloat16))
    ref = w8a8.linear(x, w)
    x2 = x.clone()
    x2[7, 100], x2[20, 0] = float("nan"), float("-inf")
    y = w8a8.linear(x2, w)
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(y[keep], ref[keep]) and bool(y[[7, 20]].isnan().all())
    x2[7] = 0
    assert not w8a8.linear(x2, w)[7].any()


@pytest.mark.parametrize("rows,K,Nn", [(1, 64, 40), (1, 7168, 4096), (2, 2048, 264), (3, 1424, 136), (4, 7168, 264),
                                       (5, 7168, 128), (17, 512, 128), (130, 512, 264), (3000, 256, 4096)])
def test_linear(rows, K, Nn):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, K, generator=g, device="cuda").to(torch.bfloat16)
    w = w8a8.quantize_weights(torch.randn(1, K, Nn, generator=g, device="cuda"))
    q, s = quant_ref(x)
    ref = product_ref(q, s, w.q, w.scale, [rows])
    got = w8a8.linear(x, w)
    assert bool(((got.double() - ref).abs() <= ref.abs() * (HALF + 2.0 ** -20)).all())


def layer_ref(x, ids, vals, w13, w2, first):
    """(y, tolerance).  A value of h may land one step off where its quotient
    is nearer to a tie than fp32 arithmetic can tell."""
    El, H, F = w2.q.shape
    y = torch.zeros(x.shape[0], H, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    q, s = quant_ref(x)
    xd = q.double() * s.double()[:, None]
    for t in range(x.shape[0]):
        seen = set()
        for k, i in enumerate(ids[t].tolist()):
            e = i - first
            if not 0 <= e < El or i in seen:
                continue
            seen.add(i)
            a = (w13.q[e].double() * w13.scale[e].double()[:, None]) @ xd[t]
            h, dh = glu_ref(a[None])
            h, dh = h[0], dh[0]
            top = h.abs().max()
            rel = float(dh.max() / top) + 2.0 ** -22 if float(top) > 0 else 0.0
            scale = (top.float() * RECIP).double()
            quot = torch.where(scale > 0, h / scale, torch.zeros_like(h))
            hq = quot.round().clamp(-127, 127)
            near = ((quot - quot.floor()) - 0.5).abs() <= quot.abs() * rel + dh / scale.clamp_min(1e-300) + 1e-12
            wd = w2.q[e].double() * w2.scale[e].double()[:, None]
            o = wd @ (hq * scale)
            v = float(vals[t, k])
            y[t] += v * o
            tol[t] += abs(v) * (wd.abs() @ ((near.double() + hq.abs() * rel) * scale) + o.abs() * 2.0 ** -20)
    return y, tol * (1 + HALF) + y.abs() * HALF + 1e-30


LAYERS = [
    # T, H, El, E, first, K, F
    (1, 64, 4, 4, 0, 1, 32),
    (1, 7168, 12, 12, 0, 8, 2048),
    (1, 512, 6, 12, 3, 16, 176),
    (1, 2048, 3, 3, 0, 2, 24576),     # h quantised by a launch of its own
    (2, 24576, 4, 4, 0, 2, 64),       # x, too
    (4, 336, 3, 3, 0, 3, 144),
    (5, 256, 2, 2, 0, 2, 128),
    (8, 1040, 2, 2, 0, 2, 96),
    (16, 256, 8, 10, 1, 1, 80),
    (17, 256, 2, 4, 1, 1, 80),
    (4, 2048, 20, 20, 0, 8, 1408),
    (32, 272, 16, 20, 1, 1, 112),
    (33, 272, 3, 5, 1, 1, 112),
    (3, 144, 8, 8, 0, 2, 112),
    (40, 256, 8, 32, 16, 6, 208),
    (65, 512, 16, 16, 0, 4, 384),
    (300, 1024, 4, 4, 0, 2, 640),
]


@pytest.mark.parametrize("T,H,El,E,first,K,F", LAYERS)
def test_layer(T, H, El, E, first, K, F):
    g = torch.Generator(device="cuda").manual_seed(T + H)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = w8a8.quantize_weights(0.05 * torch.randn(El, H, 2 * F, generator=g, device="cuda"))
    w2 = w8a8.quantize_weights(0.05 * torch.randn(El, F, H, generator=g, device="cuda"))
    ids = torch.rand(T, max(E, K), generator=g, device="cuda").topk(K, dim=-1).indices
    vals = torch.randn(T, K, generator=g, device="cuda").softmax(-1)
    if K > 1:
        ids[0, 1] = ids[0, 0]        # repeated
        ids[-1, 0] = first + El + 3  # elsewhere
        if T > 2:
            ids[1] = -1
    for dt, vt in ((torch.int64, torch.float32), (torch.int32, torch.bfloat16)):
        i, v = ids.to(dt), vals.to(vt)
        y = w8a8.moe_layer(x, i, v, w13, w2, first_expert=first)
        torch.cuda.synchronize()
        ref, tol = layer_ref(x, i, v, w13, w2, first)
        err = (y.double() - ref).abs()
        assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()}, worst {float((err / tol).max()):.2f}x"
        assert torch.equal(y, w8a8.moe_layer(x, i, v, w13, w2, first_expert=first))
    if K > 1 and T > 2:
        assert not y[1].any()


MIXED = [
    # T, H, El, E, first, K, F
    (4, 4096, 8, 16, 4, 2, 14336),    # gate and up by rows, gathered and quantised in place; down by tiles
    (1, 2048, 64, 64, 0, 8, 16384),   # the same, every row live
    (4, 2048, 32, 32, 0, 8, 4096),    # gathered and quantised by a launch of its own, multiplied by rows
    (4, 32768, 4, 6, 1, 2, 128),      # gate and up by tiles; down by rows, h quantised in place
    (24, 4112, 12, 14, 1, 1, 2048),   # the same, h quantised by a launch of its own
]


@pytest.mark.parametrize("none", [False, True])
@pytest.mark.parametrize("T,H,El,E,first,K,F", MIXED)
def test_layer_of_both_forms(T, H, El, E, first, K, F, none):
    """Sizes at which one product of the layer takes the form for a few rows
    and the other one tiles, with rows for experts elsewhere (the live rows
    end before the last) and without any live row."""
    g = torch.Generator(device="cuda").manual_seed(T + F)

    def weights(Nn, K8):
        q = torch.randint(-127, 128, (El, Nn, K8), generator=g, device="cuda", dtype=torch.int8)
        return w8a8.QuantWeights(q, (0.5 + torch.rand(El, Nn, generator=g, device="cuda")) * 2.0 ** -11)

    w13, w2 = weights(2 * F, H), weights(H, F)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1).indices
    vals = torch.randn(T, K, generator=g, device="cuda").softmax(-1)
    if none:
        ids += first + El
    elif El < E:
        ids[-1, 0] = first + El
    y = w8a8.moe_layer(x, ids, vals, w13, w2, first_expert=first)
    if none:
        assert not y.any()
        return
    ref, tol = layer_ref(x, ids, vals, w13, w2, first)
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()}, worst {float((err / tol).max()):.2f}x"
    assert torch.equal(y, w8a8.moe_layer(x, ids, vals, w13, w2, first_expert=first))


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
@pytest.mark.parametrize("first", [0, 5, 2 ** 31 - 3])
def test_layer_ids_at_the_types_ends(T, dt, first):
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, 64, generator=g, device="cuda").to(torch.bfloat16)
    w13 = w8a8.quantize_weights(0.05 * torch.randn(3, 64, 64, generator=g, device="cuda"))
    w2 = w8a8.quantize_weights(0.05 * torch.randn(3, 32, 64, generator=g, device="cuda"))
    ends = torch.iinfo(dt)
    ids = torch.tensor([ends.min, ends.max, first - 1, first, first + 1, -first], device="cuda").clamp(
        ends.min, ends.max).to(dt).expand(T, 6).contiguous()
    ids[1:] = ids[1:].roll(1, 1)
    vals = torch.rand(T, 6, generator=g, device="cuda")
    y = w8a8.moe_layer(x, ids, vals, w13, w2, first_expert=first)
    ref, tol = layer_ref(x, ids, vals, w13, w2, first)
    assert bool(((y.double() - ref).abs() <= tol).all())


def test_misaligned_and_misplaced_tensors_are_refused():
    xq, xs, wq, ws = make(5, 64, 32, 2, 1)
    cd = torch.tensor([2, 3], dtype=torch.int32, device="cuda")
    w = w8a8.QuantWeights(wq, ws)
    flat = torch.zeros(5 * 64 + 16, dtype=torch.int8, device="cuda")
    with pytest.raises(N.MoeEpError):
        w8a8.grouped_gemm(flat[1:1 + 5 * 64].view(5, 64), xs, w, cd)
    for bad in (w8a8.QuantWeights(wq, ws.cpu()), w8a8.QuantWeights(wq.cpu(), ws),
                w8a8.QuantWeights(wq.transpose(1, 2).contiguous().transpose(1, 2), ws)):
        with pytest.raises(ValueError):
            w8a8.grouped_gemm(xq, xs, bad, cd)
    with pytest.raises(ValueError):
        w8a8.grouped_gemm(xq, xs.cpu(), w, cd)
    with pytest.raises(ValueError):
        w8a8.grouped_gemm(xq, xs, w, cd.cpu())
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda")
    ids, vals = torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.ones(3, 1, device="cuda")
    w2 = w8a8.QuantWeights(torch.zeros(2, 64, 16, dtype=torch.int8, device="cuda"), torch.ones(2, 64, device="cuda"))
    w8a8.moe_layer(x, ids, vals, w, w2)
    for bad in (dict(w2=w8a8.QuantWeights(w2.q, w2.scale.cpu())), dict(top_vals=vals.cpu()), dict(first_expert=-1),
                dict(top_idxs=ids[:2]), dict(x=x[:, :32]), dict(top_vals=vals.double())):
        with pytest.raises((ValueError, TypeError)):
            w8a8.moe_layer(**{**dict(x=x, top_idxs=ids, top_vals=vals, w13=w, w2=w2), **bad})


@pytest.mark.parametrize("T", [2, 40])
def test_scales_at_any_float(T):
    """Scales need no more than a float's alignment, for any number of tokens."""
    g = torch.Generator(device="cuda").manual_seed(T)
    El, H, K, F = 3, 256, 2, 128
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = w8a8.quantize_weights(0.05 * torch.randn(El, H, 2 * F, generator=g, device="cuda"))
    w2 = w8a8.quantize_weights(0.05 * torch.randn(El, F, H, generator=g, device="cuda"))

    def odd(w):
        flat = torch.zeros(w.scale.numel() + 1, device="cuda")
        flat[1:] = w.scale.flatten()
        return w8a8.QuantWeights(w.q, flat[1:].view(w.scale.shape))

    assert odd(w13).scale.data_ptr() % 16 == 4
    ids = torch.rand(T, El, generator=g, device="cuda").topk(K, dim=-1).indices
    vals = torch.rand(T, K, generator=g, device="cuda")
    y = w8a8.moe_layer(x, ids, vals, w13, w2)
    assert torch.equal(w8a8.moe_layer(x, ids, vals, odd(w13), odd(w2)), y)
    for rows, counts in ((5, [2, 0, 3]), (330, [200, 0, 130]), (9000, [4000, 2000, 3000])):
        xq = torch.randint(-127, 128, (rows, H), generator=g, device="cuda", dtype=torch.int8)
        xs = torch.rand(rows + 1, generator=g, device="cuda")
        cd = torch.tensor(counts, dtype=torch.int32, device="cuda")
        for glu in (False, True):
            ref = w8a8.grouped_gemm(xq, xs[1:].clone(), w13, cd, swiglu=glu)
            assert torch.equal(w8a8.grouped_gemm(xq, xs[1:], odd(w13), cd, swiglu=glu), ref)


def test_layer_captured_and_on_streams():
    g = torch.Generator(device="cuda").manual_seed(6)
    T, H, E, K, F = 24, 256, 8, 2, 128
    w13 = w8a8.quantize_weights(0.05 * torch.randn(E, H, 2 * F, generator=g, device="cuda"))
    w2 = w8a8.quantize_weights(0.05 * torch.randn(E, F, H, generator=g, device="cuda"))
    vals = torch.full((T, K), 0.5, device="cuda")
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1).indices
    w8a8.moe_layer(x, ids, vals, w13, w2, first_expert=0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(w8a8.moe_layer(x, ids, vals, w13, w2))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        x.copy_(torch.randn(T, H, generator=g, device="cuda"))
        ids.copy_(torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1).indices)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        eager = w8a8.moe_layer(x, ids, vals, w13, w2)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)


def test_kernels_with_grid_barriers_side_by_side():
    """The decode layer, an 8-bit product split over K and one of whole tiles
    on three streams at once: each has the result that it has alone."""
    g = torch.Generator(device="cuda").manual_seed(11)
    T, H, E, K, F = 20, 1024, 16, 4, 512
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    w13 = (0.05 * torch.randn(E, H, 2 * F, generator=g, device="cuda")).to(torch.bfloat16)
    w2 = (0.05 * torch.randn(E, F, H, generator=g, device="cuda")).to(torch.bfloat16)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=-1).indices
    vals = torch.rand(T, K, generator=g, device="cuda")
    split = make(100, 7168, 512, 2, 12)     # two tiles of rows, two of channels: shares of K
    whole = make(9000, 512, 4096, 1, 13)    # enough tiles for every SM
    counts = torch.tensor([61, 39], dtype=torch.int32, device="cuda")
    calls = [lambda: decode.moe_layer(x, ids, vals, w13, w2),
             lambda: w8a8.grouped_gemm(*split[:2], w8a8.QuantWeights(*split[2:]), counts),
             lambda: w8a8.grouped_gemm(*whole[:2], w8a8.QuantWeights(*whole[2:]))]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(8):
        got = [[] for _ in calls]
        for _ in range(3):
            for c, s, o in zip(calls, streams, got):
                with torch.cuda.stream(s):
                    o.append(c())
        torch.cuda.synchronize()
        for w, o in zip(want, got):
            assert all(torch.equal(a, w) for a in o)


@pytest.mark.parametrize("T", [1, 6, 40])
def test_a_decode_step_with_both_operators(T):
    """As a model would run them, in one captured step: the bf16 layer routes
    its tokens, the 8-bit layer of the next block follows the same routing,
    a dense 8-bit projection comes last."""
    g = torch.Generator(device="cuda").manual_seed(T)
    H, E, K, F, Nn = 512, 16, 4, 256, 264
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    rw = (torch.randn(H, E, generator=g, device="cuda") / H ** 0.5).to(torch.bfloat16)
    w13 = (0.05 * torch.randn(E, H, 2 * F, generator=g, device="cuda")).to(torch.bfloat16)
    w2 = (0.05 * torch.randn(E, F, H, generator=g, device="cuda")).to(torch.bfloat16)
    q13, q2 = w8a8.quantize_weights(w13), w8a8.quantize_weights(w2)
    head = w8a8.quantize_weights(torch.randn(1, H, Nn, generator=g, device="cuda"))

    def step():
        y, vals, ids = decode.routed_layer(x, rw, K, w13, w2, renormalize=True)
        z = w8a8.moe_layer(y, ids, vals, q13, q2)
        return y, vals, ids, z, w8a8.linear(z, head)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        x.copy_(torch.randn(T, H, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        y, vals, ids, z, logits = out
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
        ref, tol = layer_ref(y, ids, vals, q13, q2, 0)
        assert bool(((z.double() - ref).abs() <= tol).all())
        q, s = quant_ref(z)
        ref = product_ref(q, s, head.q, head.scale, [T])
        assert bool(((logits.double() - ref).abs() <= ref.abs() * (HALF + 2.0 ** -20)).all())


@pytest.mark.parametrize("rows", [1, 20, 600])
def test_status_word_stays_clear(rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 256, generator=g, device="cuda").to(torch.bfloat16)
    w = w8a8.quantize_weights(torch.randn(1, 256, 512, generator=g, device="cuda"))
    status = torch.zeros(1, dtype=torch.int32, pin_memory=True)
    assert torch.equal(w8a8.linear(x, w, status=status), w8a8.linear(x, w))
    w8a8.grouped_gemm(*w8a8.quantize_rows(x), w, status=status)
    torch.cuda.synchronize()
    assert int(status[0]) == 0


def test_weighted_sum_uses_the_routing():
    g = torch.Generator(device="cuda").manual_seed(8)
    T, E, K, H = 50, 6, 3, 72
    ids = torch.randint(-1, E + 1, (T, K), generator=g, device="cuda")
    vals = torch.rand(T, K, generator=g, device="cuda")
    r = utils.route(ids, E, with_slots=True)
    rows = torch.randn(T * K, H, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    N.check(N.lib().moe_weighted_sum(rows.data_ptr(), 0, ids.data_ptr(), 1, 0, vals.data_ptr(), 0, r.slots.data_ptr(),
                                     r.offsets.data_ptr(), T, K, H, E, y.data_ptr(), None), "moe_weighted_sum")
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(ref)
    for t in range(T):
        for k in range(K):
            if int(r.slots[t, k]) >= 0:
                row = rows[int(r.offsets[int(ids[t, k])]) + int(r.slots[t, k])].double()
                ref[t] += float(vals[t, k]) * row
                mag[t] += float(vals[t, k]) * row.abs()
    assert bool(((y.double() - ref).abs() <= ref.abs() * HALF + mag * (K + 1) * 2.0 ** -23).all())
