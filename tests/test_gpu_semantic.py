"""The semantic head's operators on the GPU against their definitions in 64 bits (tests/semantic_ref.py derives the bounds)."""
import math

import pytest
import torch

import semantic_ref as S
from fusionsense_amd import losses, ops, scenes
from fusionsense_amd.fusion import render_fusionsense
from fusionsense_amd.semantics import SemanticHead

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def _randn(dev, *shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(dev)


def _layer(dev, M, K, N, dtype, bias=True, res=True, seed=0):
    x = _randn(dev, M, K, seed=seed, dtype=dtype)
    w = _randn(dev, N, K, seed=seed + 1).div(math.sqrt(K)).to(dtype)
    b = _randn(dev, N, seed=seed + 2, dtype=dtype) if bias else None
    r = _randn(dev, M, N, seed=seed + 3, dtype=dtype) if res else None
    dy = _randn(dev, M, N, seed=seed + 4, dtype=dtype)
    return x, w, b, r, dy


def _check_layer(x, w, b, r, act, dy, what=""):
    leaves = {k: t.detach().requires_grad_(True) for k, t in (("x", x), ("w", w), ("b", b), ("r", r)) if t is not None}
    y = ops.linear_act(leaves["x"], leaves["w"], leaves.get("b"), act, leaves.get("r"))
    assert y.dtype == x.dtype and y.shape == x.shape[:-1] + (w.shape[0],)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    K, N = x.shape[-1], w.shape[0]
    want = S.linear(x.reshape(-1, K), w, b, r.reshape(-1, N) if r is not None else None, act, dy.reshape(-1, N))
    S.check(y.reshape(-1, N), want["y"], f"{what} y")
    S.check(grads["x"].reshape(-1, K), want["dx"], f"{what} dx")
    S.check(grads["w"], want["dw"], f"{what} dw")
    if b is not None:
        S.check(grads["b"], want["db"], f"{what} db")
    if r is not None:
        assert torch.equal(grads["r"], dy)
    return y, grads


SIZES = [(1, 1, 1), (1, 64, 150), (2, 3, 5), (7, 31, 33), (64, 64, 64), (127, 33, 65), (129, 128, 128), (300, 130, 257),
         (1000, 32, 150), (33, 513, 40), (65, 257, 768), (5, 1024, 1500), (2500, 16, 7), (4097, 96, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_linear_sizes(dev, size, dtype):
    i = SIZES.index(size)
    act = list(ops.ACTIVATIONS)[i % 4]
    _check_layer(*_layer(dev, *size, dtype, bias=i % 3 != 0, res=i % 2 == 0, seed=i)[:4], act,
                 _layer(dev, *size, dtype, seed=i)[4], f"{size} {act}")


@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_activations(dev, act, dtype):
    for bias, res in ((True, True), (False, False), (True, False), (False, True)):
        x, w, b, r, dy = _layer(dev, 200, 64, 72, dtype, bias, res, seed=5)
        _check_layer(x * 3, w, b, r, act, dy, f"{act} {bias} {res}")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_layouts(dev, dtype):
    """Slices of wider planes, rows of an odd pitch, unaligned starts, expanded rows, transposed inputs, leading axes."""
    M, K, N = 150, 40, 24
    x, w, b, r, dy = _layer(dev, M, K, N, dtype, seed=9)
    y0, g0 = _check_layer(x, w, b, r, "gelu", dy)
    wide = torch.full((M, K + 3), float("nan"), dtype=dtype, device=dev)
    wide[:, 1:K + 1] = x
    rw = torch.full((M, N + 1), float("nan"), dtype=dtype, device=dev)
    rw[:, 1:] = r
    for xx, rr, gg in ((wide[:, 1:K + 1], rw[:, 1:], dy), (x.t().contiguous().t(), r.t().contiguous().t(), dy.t().contiguous().t())):
        y, g = _check_layer(xx, w, b, rr, "gelu", gg, "layout")
        assert torch.equal(y, y0) and all(torch.equal(g[k], g0[k]) for k in ("x", "w", "b"))
    wt = w.t().contiguous().t()  # (a weight that is a transposed view)
    y, g = _check_layer(x, wt, b, r, "gelu", dy, "weight view")
    assert torch.equal(y, y0)
    y, g = _check_layer(x.reshape(3, 5, 10, K), w, b, r.reshape(3, 5, 10, N), "gelu", dy.reshape(3, 5, 10, N), "leading axes")
    assert torch.equal(y.reshape(M, N), y0)
    # one row for all: its gradient is the sum over the rows (torch's, over the operator's)
    row, rrow = x[:1].clone().requires_grad_(True), r[:1].clone().requires_grad_(True)
    y = ops.linear_act(row.expand(M, K), w, b, "silu", rrow.expand(M, N))
    want = S.linear(x[:1].expand(M, K), w, b, r[:1].expand(M, N), "silu", torch.ones(M, N))
    S.check(y, want["y"], "expanded y")
    y.sum().backward()  # (dy: one value expanded over both axes)
    v, e = want["dx"]
    ulp = S.U[dtype] * v.sum(0).abs() * 2 + M * S.U32 * v.abs().sum(0)
    S.check(row.grad[0], (v.sum(0), e.sum(0) + ulp + S.TINY[dtype]), "expanded dx")
    assert torch.equal(rrow.grad, torch.full_like(rrow, M))
    # a single feature vector without a row axis
    S.check(ops.linear_act(x[0], w, b)[None], S.linear(x[:1], w, b, None, "none")["y"], "vector")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("only", ["x", "w", "b", "r"])
def test_linear_single_gradients(dev, only, dtype):
    """Each gradient alone is the one that comes with the others, bit for bit."""
    x, w, b, r, dy = _layer(dev, 333, 48, 96, dtype, seed=2)
    _, g0 = _check_layer(x, w, b, r, "silu", dy)
    t = {"x": x, "w": w, "b": b, "r": r}
    t[only] = t[only].detach().requires_grad_(True)
    g, = torch.autograd.grad(ops.linear_act(t["x"], t["w"], t["b"], "silu", t["r"]), [t[only]], dy)
    assert torch.equal(g, g0[only])


def test_linear_without_rows(dev):
    x = torch.zeros(0, 5, device=dev, requires_grad=True)
    w = torch.ones(4, 5, device=dev, requires_grad=True)
    b = torch.ones(4, device=dev, requires_grad=True)
    y = ops.linear_act(x, w, b, "relu", torch.zeros(0, 4, device=dev))
    assert y.shape == (0, 4)
    y.sum().backward()
    assert x.grad.shape == (0, 5) and not w.grad.any() and not b.grad.any()


def test_linear_refuses(dev):
    x, w, b, r, _ = _layer(dev, 4, 8, 6, torch.float32)
    for args in ((x, w.half()), (x, w, b.half()), (x, w, b, "none", r.half()), (x, w, b, "tanh"), (x, w[:, :7]), (x, w[0]),
                 (x, w, b[:5]), (x, w, b, "none", r[:3]), (x, w, b, "none", r[0]), (x, w.cpu()), (x, torch.zeros(0, 8, device=dev)),
                 (torch.zeros((), device=dev), w)):
        with pytest.raises(ValueError):
            ops.linear_act(*args)
    x.requires_grad_(True)
    y = ops.linear_act(x, w, b, "silu")
    g, = torch.autograd.grad(y, [x], torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_keeps_bad_values_in_their_rows(dev, dtype):
    x, w, b, r, dy = _layer(dev, 200, 64, 64, dtype, seed=3)
    y0 = ops.linear_act(x, w, b, "relu", r)
    x2 = x.clone()
    x2[17, 3], x2[130, 60], x2[199, 0] = float("nan"), float("inf"), -float("inf")
    y2 = ops.linear_act(x2, w, b, "relu", r)
    keep = torch.ones(200, dtype=torch.bool, device=dev)
    keep[[17, 130, 199]] = False
    assert torch.equal(y2[keep], y0[keep])
    assert torch.isnan(y2[17]).all()
    assert torch.equal(y2[130], torch.where(w[:, 60] > 0, torch.full_like(r[130], float("inf")), r[130]))


# A layer per kernel that forms dz: few values, one pass, few rows, rows, tiles of 64 and of 128 rows.
DZ = [(3, 7, 5), (300, 64, 72), (40, 2000, 1100), (1100, 8, 400), (3000, 300, 70), (2200, 600, 130), (2200, 2100, 1100)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("res", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("size", DZ, ids=lambda s: "x".join(map(str, s)))
def test_linear_relu_drops_gradients_of_what_it_cut_off(dev, dtype, res, size):
    """Infinite and NaN gradients where the pre-activation is clearly negative: the bits that zeros there give."""
    x, w, b, r, dy = _layer(dev, *size, dtype, res=res, seed=64)
    z = x.float() @ w.float().t() + b.float()
    cut = (z < -0.1) & (torch.rand(z.shape, generator=torch.Generator().manual_seed(65)).to(dev) < 0.2)
    bad = torch.tensor([math.inf, -math.inf, math.nan], device=dev)[torch.arange(z.numel(), device=dev).reshape(z.shape) % 3].to(dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    y = ops.linear_act(*leaves, "relu", r)
    want = torch.autograd.grad(y, leaves, dy.masked_fill(cut, 0), retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch.where(cut, bad, dy))
    assert cut.any() and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("res", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("size", DZ, ids=lambda s: "x".join(map(str, s)))
def test_linear_relu_slope_of_values_that_round_to_zero(dev, size, res):
    """fp16: a pre-activation of 2^-26 or 2^-25 has slope one though the output is zero, one of 0 or -2^-26 has none; alike in
    every kernel.  (Column n of x picks row n's weight: one term a sum, exact.)"""
    M, K, N = size
    dtype = torch.float16
    x, w, dy = torch.zeros(M, K, dtype=dtype), torch.zeros(N, K, dtype=dtype), _randn("cpu", M, N, seed=66, dtype=dtype)
    x[:, 0] = 2.0 ** -13
    values = torch.tensor([2.0 ** -13, 2.0 ** -12, 0.0, -(2.0 ** -13), 1.5 * 2.0 ** -12, 1.0])
    w[:, 0] = values[torch.arange(N) % 6].to(dtype)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, torch.zeros(N, dtype=dtype))]
    r = torch.zeros(M, N, dtype=dtype, device=dev) if res else None
    y = ops.linear_act(*leaves, "relu", r)
    z = x[0, 0].double() * w[:, 0].double()
    assert torch.equal(y.detach().cpu(), z.clamp(min=0).to(dtype).expand(M, N)) and (z > 0).sum() > (y[0] != 0).sum()
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(dev))
    dz = dy.double() * (z > 0)
    for got, v, mag in ((dx, dz @ w.double(), dz.abs() @ w.double().abs()), (dw, dz.t() @ x.double(), dz.abs().t() @ x.double().abs()),
                        (db, dz.sum(0), dz.abs().sum(0))):
        e = (max(M, N) + 2) * S.U32 * mag
        S.check(got, (v, e + S.U[dtype] * (v.abs() + e) + S.TINY[dtype]), "")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_activation_over_its_range(dev, dtype, act):
    """act and its slope of single numbers over [-14, 14] (one term a sum: z is exact).

    gelu's tail h = P(t) exp(-z^2/2) is off by its fit, 1.3e-9, and relatively by the exponent's rounding, z^2 / 2 times two
    roundings, and by 32 U32 for P (seven steps, magnitudes 2.7 times the sum), the reciprocal and the exponential; bf16's form by
    1e-4; fp16's by 5.6e-6 and, for |z| <= 6, by 72 U32 (one rounding a step of Q's evaluation: their magnitudes sum to 100, ln 2
    of which is h's, and the exponential's two), by 2^-26 beyond.  y = max(z, 0) - |z| h; the slope is h - |z| phi, or one minus
    that.  silu's sigma is off by (2 |z| + 8) U32 of itself.  The type's rounding comes last; dz enters its product as two values of a half-width type."""
    z = torch.linspace(-14, 14, 100000).to(dtype)
    x = z[:, None].to(dev).requires_grad_(True)
    y = ops.linear_act(x, torch.ones(1, 1, dtype=dtype, device=dev), None, act)
    dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    z = z.double()
    u, size = S.U[dtype], z.abs()
    if act == "gelu":
        h, phi = 0.5 * torch.erfc(size / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        rel = (z * z + 32) * S.U32
        # (the exponential instruction gives zero for what lies below 2^-126, bf16's tail from |z| = 13.1 on: off by that at most)
        ey = size * {torch.float32: 1.3e-9 + rel * h, torch.bfloat16: 1e-4 * h + 2.0 ** -126,
                     torch.float16: (5.6e-6 + 72 * S.U32) * h}[dtype]
        if dtype == torch.float16:
            ey = ey + 2.0 ** -26 * (size > 6)
        es = 1.3e-9 + rel * (h + size * phi) + 2 * S.U32
        low = 0.5 * torch.erfc(-z / math.sqrt(2))  # (1 + erf, as S has it, is 2e-16 off: all of the value at z = -9)
        vy, vs = z * low, low + z * phi
    else:
        rel = (2 * size + 8) * S.U32
        ey = rel * size * torch.sigmoid(z)
        es = 2 * rel * torch.sigmoid(z) * (1 + size) + 2 * S.U32
        vy, vs = S.act(z, act), S.slope(z, act)
    for got, v, e in ((y, vy, ey), (dx, vs, es)):
        e = e + 2 * S.U32 * v.abs() + (u * u * v.abs() + S.TINY[dtype] if got is dx and dtype != torch.float32 else 0)
        S.check(got, (v[:, None], (e + u * (v.abs() + e) + S.TINY[dtype])[:, None]), "y" if got is y else "dx")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("K", [64, 700])
def test_linear_infinite_pre_activations(dev, dtype, act, K):
    """What z Phi(z) and z sigma(z) give: +inf stays, -inf and NaN become NaN, the largest finite sums stay or vanish."""
    x = torch.zeros(3000, K, dtype=dtype, device=dev)
    big = torch.finfo(dtype).max
    values = [float("inf"), -float("inf"), float("nan"), big, -big]
    x[40:45, 1] = torch.tensor(values, dtype=dtype, device=dev)
    w = torch.zeros(70, K, dtype=dtype, device=dev)
    w[:, 1] = 1
    y = ops.linear_act(x, w, None, act)
    want = [float("inf"), float("nan"), float("nan"), big, 0.0]
    for m, v in enumerate(want):
        assert torch.equal(y[40 + m].isnan(), torch.full_like(y[0], v).isnan())
        assert v != v or (y[40 + m].abs() == abs(v)).all()
    assert not y[:40].any() and not y[45:].any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("K", [24, 64, 200, 700])
@pytest.mark.parametrize("pitch", [1, 3, 8])
def test_linear_overlapping_rows(dev, dtype, K, pitch):
    """Sliding windows over one vector (rows closer together than they are long), forward and backward."""
    M, N = 300, 70
    v = _randn(dev, (M - 1) * pitch + K, seed=80, dtype=dtype)
    x = v.as_strided((M, K), (pitch, 1))
    x0, w, b, r, dy = _layer(dev, M, K, N, dtype, seed=81)
    y0, g0 = _check_layer(x.clone(), w, b, r, "gelu", dy)
    g = _randn(dev, (M - 1) * pitch + N, seed=82, dtype=dtype).as_strided((M, N), (pitch, 1))
    leaves = [t.detach().requires_grad_(True) for t in (w, b)]
    out = ops.linear_act(x, leaves[0], leaves[1], "gelu", r)
    got = torch.autograd.grad(out, leaves, dy)
    assert torch.equal(out, y0) and torch.equal(got[0], g0["w"]) and torch.equal(got[1], g0["b"])
    _check_layer(x.clone(), w, b, r, "silu", g, "windows of gradients")


def test_linear_gradients_against_differences(dev):
    """fp32, central differences of sum(dy * y) along random directions.  y carries (K + 2) U32 of its terms (S.linear's bound);
    with a step h the quotient is off by that over h plus h^2 / 6 times the third derivative along the direction (act''' <= 2
    for gelu and silu: |z'|^3 * 2)."""
    for act in ("gelu", "silu", "none"):
        x, w, b, r, dy = _layer(dev, 40, 24, 20, torch.float32, seed=11)
        _, g = _check_layer(x, w, b, r, act, dy)
        h = 2.0 ** -6
        for name, t in (("x", x), ("w", w), ("b", b)):
            d = _randn(dev, *t.shape, seed=12) / math.sqrt(t.shape[-1])
            val, err, zd = [], 0.0, None
            for s in (h, -h):
                a = {"x": x, "w": w, "b": b}
                a[name] = t + s * d
                val.append(float((ops.linear_act(a["x"], a["w"], a["b"], act, r).double() * dy.double()).sum()))
                # (the moved input as it was rounded: its own rounding shifts z by U32 of its size)
                bound = S.linear(a["x"], a["w"], a["b"], r, act)["y"][1]
                err += float((bound * dy.cpu().double().abs()).sum())
                z = a["x"].double().abs() @ a["w"].double().abs().t() + a["b"].double().abs()
                err += float((1.13 * S.U32 * z * dy.double().abs()).sum())
            zd = {"x": lambda: d.double() @ w.double().t(), "w": lambda: x.double() @ d.double().t(),
                  "b": lambda: d.double().expand(40, 20)}[name]()
            third = 0.0 if act == "none" else float((2 * zd.abs() ** 3 * dy.double().abs()).sum()) * h * h / 6
            quotient = (val[0] - val[1]) / (2 * h)
            want = float((g[name].double() * d.double()).sum())
            assert abs(quotient - want) <= err / (2 * h) + third + 1e-5 * abs(want), (act, name, quotient, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16], ids=["bf16"])
def test_linear_offsets_beyond_32_bits(dev, dtype):
    """Rows 2^21 + 1 elements apart over more than 2^31 elements, and an output of more than 2^31 elements."""
    M, K, N, pitch = 1100, 24, 16, (1 << 21) + 1
    big = torch.empty(M * pitch, dtype=dtype, device=dev)
    assert big.numel() > 2 ** 31
    x0, w, b, _, dy = _layer(dev, M, K, N, dtype, seed=21)
    x = big.as_strided((M, K), (pitch, 1))
    x.copy_(x0)
    y0, g0 = _check_layer(x0, w, b, None, "gelu", dy)
    y, g = _check_layer(x, w, b, None, "gelu", dy)
    assert torch.equal(y, y0) and all(torch.equal(g[k], g0[k]) for k in g0)
    del big, x
    M, N = (1 << 31) // 1500 + 77, 1500
    x = _randn(dev, 4096, 8, seed=22, dtype=dtype).repeat((M + 4095) // 4096, 1)[:M]
    w, b = _randn(dev, N, 8, seed=23, dtype=dtype), _randn(dev, N, seed=24, dtype=dtype)
    y = ops.linear_act(x, w, b, "relu")
    first = y[:4096]
    S.check(first[:64], S.linear(x[:64], w, b, None, "relu")["y"], "first rows")
    for m0 in range(0, M, 4096 * 64):
        n = min(4096 * 64, M - m0)
        blk = y[m0:m0 + n]
        assert torch.equal(blk, first.repeat((n + 4095) // 4096, 1)[:n]), m0


# Sizes at which the product, its dz, dx and dW take other kernels or tiles than above: many tiles of 128 and of 64 columns, a last
# tile of two columns, a last slab of a few entries, few rows of a long sum, more than 256 outputs of a short one, dW tiles of
# either shape, several slices and a single one.
WIDE = [(3000, 300, 70), (7000, 200, 50), (2200, 600, 130), (1290, 161, 513), (130, 48, 300), (1500, 200, 64), (16, 1100, 33),
        (1100, 8, 400), (40, 2000, 1100), (129, 64, 257), (3000, 96, 900)]


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", WIDE, ids=lambda s: "x".join(map(str, s)))
def test_linear_wide_sizes(dev, size, dtype, act):
    i = WIDE.index(size)
    x, w, b, r, dy = _layer(dev, *size, dtype, bias=i % 3 != 1, res=act == "silu", seed=30 + i)
    _check_layer(x, w, b, r, act, dy, f"{size} {act}")


FEW = [(1, 1, 1), (1, 3, 2), (2, 1, 3), (1, 40, 500), (16, 64, 20), (17, 33, 30), (512, 24, 1), (3, 1000, 170), (1, 1024, 512), (100, 7, 5),
       (8, 65, 64), (9, 64, 64)]


@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", FEW, ids=lambda s: "x".join(map(str, s)))
def test_linear_few_values(dev, size, dtype, act):
    """Few rows and outputs.  Half width, up to 512 values of dz and 2^18 weights: no rounding of dz, so dx, dW and db are off by
    half a step of their own and the fp32 sums only (the bound of a layer whose dz is exact in fp32)."""
    i = FEW.index(size)
    x, w, b, r, dy = _layer(dev, *size, dtype, bias=i % 2 == 0, res=i % 3 == 0, seed=100 + i)
    _, g = _check_layer(x, w, b, r, act, dy, f"{size} {act}")
    M, K, N = size
    if dtype == torch.float32 or M * N > 512 or K * N > 1 << 18:
        return
    f = lambda t: t.float() if t is not None else None  # noqa: E731
    want = S.linear(f(x), f(w), f(b), None, act, f(dy))  # (bounds without the rounding of dz, and with fp32's of the result)
    for k, n in (("x", "dx"), ("w", "dw"), ("b", "db")):
        if k in g:
            v, e = want[n]
            S.check(g[k], (v, e + S.U[dtype] * (v.abs() + e) + S.TINY[dtype]), f"{size} {act} {n} without a rounding of dz")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", [(5000, 8, 2), (700, 32, 32), (3000, 100, 10), (1000, 250, 4), (2000, 4, 200), (10, 20, 150), (300, 3, 129),
                                  (128, 8, 200), (129, 12, 60)], ids=lambda s: "x".join(map(str, s)))
def test_linear_few_gradient_values(dev, size, dtype, act):
    """Thin layers (128 inputs at most) with a thousand values of dW, or of dx, or fewer: their products take dz as two values of
    the type, so they are off by half a step of their own, half a step of half a step of dz, and the fp32 sums.  (250 inputs are
    no thin layer: the bound of every layer.)"""
    x, w, b, r, dy = _layer(dev, *size, dtype, res=False, seed=120 + size[0])
    _, g = _check_layer(x, w, b, r, act, dy, f"{size} {act}")
    if size[1] > 128:
        return
    want = S.linear(x.float(), w.float(), b.float(), None, act, dy.float())
    u = S.U[dtype]
    dz = (dy.double() * S.slope(x.double() @ w.double().t() + b.double(), act)).abs().cpu()
    left = {"dx": dz @ w.cpu().double().abs(), "dw": dz.t() @ x.cpu().double().abs()}
    for k, n in (("x", "dx"), ("w", "dw")):
        v, e = want[n]
        # (what the second value leaves: half a step of a number that is half a step of dz at most, or a least subnormal)
        e = e + u * u * left[n] + S.TINY[dtype] * (x.abs().sum(0).cpu().double() if n == "dw" else w.abs().sum(0).cpu().double())
        S.check(g[k], (v, e + u * (v.abs() + e) + S.TINY[dtype]), f"{size} {act} {n}")


def _check_two_values(size, x, w, b, act, dy, what):
    """dx, dW and db of a half-width layer whose dz goes into its products as two values of the type: half a step of their own,
    half a step of half a step of dz, and the fp32 sums."""
    _, g = _check_layer(x, w, b, None, act, dy, what)
    want = S.linear(x.float(), w.float(), b.float(), None, act, dy.float())
    u = S.U[x.dtype]
    dz = (dy.double() * S.slope(x.double() @ w.double().t() + b.double(), act)).abs().cpu()
    left = {"dx": dz @ w.cpu().double().abs(), "dw": dz.t() @ x.cpu().double().abs(), "db": 0.0}
    tiny = {"dw": x.abs().sum(0).cpu().double(), "dx": w.abs().sum(0).cpu().double(), "db": 0.0}
    for k, n in (("x", "dx"), ("w", "dw"), ("b", "db")):
        v, e = want[n]
        # (what the second value leaves: half a step of a number that is half a step of dz at most, or a least subnormal; twice
        # as many terms, so twice the fp32 sums' part)
        e = 2 * e + u * u * left[n] + S.TINY[x.dtype] * tiny[n]
        S.check(g[k], (v, e + u * (v.abs() + e) + S.TINY[x.dtype]), f"{what} {n}")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", [(5000, 64, 128), (3000, 128, 128), (4097, 33, 190), (2000, 16, 224), (600, 100, 64), (130, 128, 65),
                                  (1000, 7, 129), (2500, 64, 160), (127, 40, 100)], ids=lambda s: "x".join(map(str, s)))
def test_linear_thin_gradients_keep_dz(dev, size, dtype, act):
    x, w, b, r, dy = _layer(dev, *size, dtype, res=False, seed=140 + size[0])
    _check_two_values(size, x, w, b, act, dy, f"{size} {act}")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("size", DZ[2:] + [(7000, 200, 50), (300, 256, 64), (129, 64, 257), (16, 300, 200), (1, 300, 1000), (513, 130, 33),
                                           (70000, 32, 256), (20000, 136, 17), (17000, 136, 1024), (33000, 300, 528)], ids=lambda s: "x".join(map(str, s)))
def test_linear_wide_gradients_keep_dz(dev, size, dtype, act):
    """... of wider layers: every kernel that forms dz or takes it, one slice of the rows and several."""
    x, w, b, r, dy = _layer(dev, *size, dtype, res=False, seed=160 + size[0])
    _check_two_values(size, x, w, b, act, dy, f"{size} {act}")


def test_linear_gradients_of_very_large_weights(dev):
    """16 400 x 16 400 weights, more values than a grid has groups of 16 threads for: dx whole, dW and db by blocks of rows."""
    M, D, dtype = 3, 16400, torch.bfloat16
    assert D * D * 16 > 2 ** 32
    g = torch.Generator(device=dev).manual_seed(0)
    x, b, dy = (torch.randn(s, generator=g, device=dev).to(dtype) for s in ((M, D), (D,), (M, D)))
    w = torch.randn(D, D, generator=g, device=dev).div_(math.sqrt(D)).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_act(*leaves, "gelu"), leaves, dy)
    want, err, mag = 0, 0, 0
    for n in range(0, D, 1025):
        wn = w[n:n + 1025].detach()
        part = S.linear(x, wn, b[n:n + 1025], None, "gelu", dy[:, n:n + 1025])
        S.check(dw[n:n + 1025], part["dw"], f"dw {n}")
        S.check(db[n:n + 1025], part["db"], f"db {n}")
        v, e = part["dx"]  # (with a rounding to the type that only the whole has: the bound is the larger for it)
        want, err, mag = want + v, err + e, mag + v.abs()
    S.check(dx, (want, err + 17 * S.U32 * mag + S.U[dtype] * want.abs()), "dx")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("size", [(700, 64, 128), (300, 128, 40), (500, 300, 70)], ids=lambda s: "x".join(map(str, s)))
def test_linear_largest_fp16_gradients(dev, size, act):
    """dz beyond fp16's largest number (60 000 times a slope of 1.13): finite gradients stay finite, infinite ones do not."""
    x, w, b, r, dy = _layer(dev, *size, torch.float16, res=False, seed=150)
    x, w, b = x * 2.0 ** -9, w * 2.0 ** -4, b * 0 + 1.4  # (z = 1.4: slopes of 1.13 and 1.03)
    sign = _randn(dev, 1, size[2], seed=151).sign() * torch.where(torch.arange(size[0], device=dev) % 2 == 0, 1.0, -1.0)[:, None]
    dy = (60000.0 * sign).to(torch.float16)  # (signs alternate down a column: the sums stay in range)
    _check_two_values(size, x, w, b, act, dy, f"{size} {act}")
    dy[3, 5] = math.inf
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_act(*leaves, act), leaves, dy)
    assert not torch.isfinite(dx[3]).any() and torch.isfinite(dx[:3]).all() and torch.isfinite(dx[4:]).all()
    assert not torch.isfinite(dw[5]).any() and not torch.isfinite(db[5]) and torch.isfinite(dw[:5]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", [(300, 600, 130), (2500, 300, 140), (200, 40, 300)], ids=lambda s: "x".join(map(str, s)))
def test_linear_wide_layouts(dev, size, dtype):
    """One row for all, slices with an odd start and pitch, gradients with a pitch, of wide layers: what the plain copies give."""
    M, K, N = size
    x, w, b, r, dy = _layer(dev, M, K, N, dtype, seed=60)
    y0, g0 = _check_layer(x, w, b, None, "relu", dy)
    wide = torch.full((M, K + 3), float("nan"), dtype=dtype, device=dev)
    wide[:, 1:K + 1] = x
    gw = torch.full((M, N + 5), float("nan"), dtype=dtype, device=dev)
    gw[:, 3:N + 3] = dy
    y, g = _check_layer(wide[:, 1:K + 1], w, b, None, "relu", gw[:, 3:N + 3], "slices")
    assert torch.equal(y, y0) and all(torch.equal(g[k], g0[k]) for k in g0)
    one = x[:1].expand(M, K)
    y, _ = _check_layer(one, w, b, r[:1].expand(M, N), "gelu", dy[:1].expand(M, N), "one row for all")
    assert torch.equal(y, y[:1].expand(M, N))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("K,N", [(32, 150), (16, 21), (24, 35), (40, 43), (32, 64), (20, 9), (64, 147), (128, 150), (300, 129)])
def test_linear_large_outputs(dev, dtype, K, N):
    """Outputs beyond 32 MiB, which leave past the caches (in whole lines, through LDS, or plainly, by their rows' length): the
    first 1000 rows against 64 bits, the others, which repeat them, bit for bit; dx likewise."""
    M = (33 << 20) // (N * dtype.itemsize) + 5
    base, w, b, r, _ = _layer(dev, 1000, K, N, dtype, seed=90)
    x = base.repeat(M // 1000 + 1, 1)[:M]
    for act, res in (("none", False), ("gelu", True)):
        rr = r.repeat(M // 1000 + 1, 1)[:M] if res else None
        v, e = S.linear(base, w, b, r if res else None, act)["y"]
        y = ops.linear_act(x, w, b, act, rr)
        S.check(y[:1000], (v, e), f"first rows {act}")
        for m0 in range(0, M, 1000):
            blk = y[m0:m0 + 1000]
            assert torch.equal(blk, y[:blk.shape[0]]), (act, m0)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    dy = torch.ones(1, 1, dtype=dtype, device=dev).expand(M, N)
    dx, _, _ = torch.autograd.grad(ops.linear_act(*leaves, "silu"), leaves, dy)
    want = S.linear(base, w, b, None, "silu", torch.ones(1000, N))
    S.check(dx[:1000], want["dx"], "dx")
    for m0 in range(0, M, 1000):
        blk = dx[m0:m0 + 1000]
        assert torch.equal(blk, dx[:blk.shape[0]]), ("dx", m0)


def test_linear_rows_too_far_apart_for_32_bit_offsets(dev):
    """Tiles whose 128 rows span more than 4 GiB: the same bits as with the rows side by side."""
    M, K, N, pitch, dtype = 130, 600, 1100, 17_000_000, torch.bfloat16
    assert pitch * 2 * 128 > 2 ** 32
    x0, w, b, _, dy0 = _layer(dev, M, K, N, dtype, seed=61)
    big = torch.zeros(M * pitch, dtype=dtype, device=dev)
    x = big.as_strided((M, K), (pitch, 1))
    x.copy_(x0)
    dy = big.as_strided((M, N), (pitch, 1), 10_000)
    dy.copy_(dy0)
    y0, g0 = _check_layer(x0, w, b, None, "none", dy0)
    y, g = _check_layer(x, w, b, None, "none", dy, "far rows")
    assert torch.equal(y, y0) and all(torch.equal(g[k], g0[k]) for k in g0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_linear_writes_its_outputs_only(dev, dtype):
    """Outputs at unaligned places between guard values, through the C entries: nothing around them changes."""
    from fusionsense_amd._lib import load, ptr, stream_ptr
    for M, K, N in ((70, 40, 24), (300, 300, 130), (3, 7, 5), (130, 48, 300)):
        x, w, b, _, dy = _layer(dev, M, K, N, dtype, seed=62)
        want, g0 = _check_layer(x, w, b, None, "gelu", dy)
        lib, dt, act = load(), ops.DTYPES[dtype], ops.ACTIVATIONS["gelu"]
        n = lib.fsgs_linear_bwd_scratch_bytes(M, K, N, dt, act, 1, 1, 1)
        scratch = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device=dev)
        room = [torch.full((t.numel() + 9,), 3.0, dtype=dtype, device=dev) for t in (want, x, w, b)]
        outs = [t[3:-6] for t in room]
        at = [t.data_ptr() for t in outs]
        assert lib.fsgs_linear_fwd(M, K, N, dt, ptr(x), K, ptr(w), ptr(b), act, None, 0, at[0], stream_ptr(dev)) == 0
        assert lib.fsgs_linear_bwd(M, K, N, dt, ptr(x), K, ptr(w), ptr(b), act, None, ptr(dy), N, at[1], at[2], at[3], ptr(scratch),
                                   n, stream_ptr(dev)) == 0
        for t, o, v in zip(room, outs, (want, g0["x"], g0["w"], g0["b"])):
            assert torch.equal(o.reshape(v.shape), v)
            assert (t[:3] == 3).all() and (t[-6:] == 3).all()
        assert (scratch[n:] == 0x5A).all()
        assert lib.fsgs_linear_bwd(M, K, N, dt, ptr(x), K, ptr(w), ptr(b), act, None, ptr(dy), N, at[1], at[2], at[3], ptr(scratch),
                                   n - 1, stream_ptr(dev)) < 0  # (a workspace one byte short is refused)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("size", [(1, 256, 1024), (4, 512, 512), (16, 300, 200), (17, 300, 200), (5, 1024, 1500), (1, 256, 4096), (16, 200, 2100),
                                  (9, 2100, 1100), (33, 130, 600), (64, 129, 300)], ids=lambda s: "x".join(map(str, s)))
def test_linear_bwd_stays_inside_its_workspace(dev, dtype, act, size):
    """Few rows of wide layers, whose dz the tile kernels form: nothing behind the workspace changes, and the bias gradient, which
    is summed from it, is right."""
    from fusionsense_amd._lib import load, ptr, stream_ptr
    M, K, N = size
    x, w, b, r, dy = _layer(dev, M, K, N, dtype, seed=63)
    want, g0 = _check_layer(x, w, b, r, act, dy)
    lib, dt, code = load(), ops.DTYPES[dtype], ops.ACTIVATIONS[act]
    n = lib.fsgs_linear_bwd_scratch_bytes(M, K, N, dt, code, 1, 1, 1)
    scratch = torch.full((n + 32 * N,), 0x5A, dtype=torch.uint8, device=dev)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    assert lib.fsgs_linear_bwd(M, K, N, dt, ptr(x), K, ptr(w), ptr(b), code, None, ptr(dy), N, ptr(dx), ptr(dw), ptr(db),
                               ptr(scratch), n, stream_ptr(dev)) == 0
    assert (scratch[n:] == 0x5A).all()
    for got, k in ((dx, "x"), (dw, "w"), (db, "b")):
        assert torch.equal(got, g0[k]), k


# ---- distillation -------------------------------------------------------------------------------------------------
def _record(dev, R, V, K, dtype, tdtype=torch.float32, idx_dtype=torch.int64, seed=0, ragged=True):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(R, V, generator=g) * 2).to(dtype).to(dev)
    if K <= V:
        idx = torch.rand(R, V, generator=g).topk(K, dim=1).indices
    else:
        idx = torch.randint(0, V, (R, K), generator=g)
    top = (torch.randn(R, K, generator=g) * 2).to(tdtype)
    if ragged:
        n = torch.randint(0, K + 1, (R, 1), generator=g)
        gone = torch.arange(K)[None] >= n
        idx = idx.masked_fill(gone, -1)
        top = top.masked_fill(gone, float("nan"))  # (padding holds anything)
    return logits, idx.to(idx_dtype).to(dev), top.to(dev)


def _check_distill(logits, idx, top, T=1.0, weight=None, reduction="mean", seed=7, what=""):
    V, K = logits.shape[-1], idx.shape[-1]
    leaf = logits.detach().requires_grad_(True)
    loss = losses.topk_distill_loss(leaf, idx, top, T, weight, reduction)
    lead = logits.shape[:-1]
    assert loss.dtype == torch.float32 and loss.shape == (lead if reduction == "none" else ())
    g = _randn(logits.device, *loss.shape, seed=seed)
    grad, = torch.autograd.grad(loss, [leaf], g)
    with torch.no_grad():
        assert torch.equal(losses.topk_distill_loss(logits, idx, top, T, weight, reduction), loss) or torch.isnan(loss).any()
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    want = S.distill(logits.reshape(-1, V), idx.reshape(-1, K), top.reshape(-1, K), T,
                     weight.reshape(-1).float() if weight is not None else None, reduction, g.reshape(-1) if g.dim() else g)
    S.check(loss, want["loss"], f"{what} loss")
    S.check(grad.reshape(-1, V), want["dlogits"], f"{what} dlogits")
    return loss.detach(), grad


DSIZES = [(1, 1, 1), (1, 150, 8), (3, 2, 2), (5, 21, 4), (70, 64, 64), (257, 65, 7), (100, 150, 16), (33, 1203, 32), (9, 700, 100),
          (4, 2049, 256), (3, 9000, 64), (3, 32003, 64), (2, 40001, 5), (2, 524288, 3), (3, 8193, 9), (3, 4095, 9), (2, 33, 256), (5000, 17, 3), (20011, 5, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("size", DSIZES, ids=lambda s: "x".join(map(str, s)))
def test_distill_sizes(dev, size, dtype):
    i = DSIZES.index(size)
    logits, idx, top = _record(dev, *size, dtype, TYPES[i % 3], [torch.int64, torch.int32][i % 2], seed=i)
    weight = torch.rand(size[0], generator=torch.Generator().manual_seed(i)).to(dev) if i % 2 else None
    for reduction in ops.REDUCTIONS:
        _check_distill(logits, idx, top, (1.0, 2.0, 0.5)[i % 3], weight, reduction, what=f"{size} {reduction}")


# Rows at the boundaries between lanes per row, steps per lane and a workgroup per row: L lanes hold 3 or 5 chunks of 4 or 8 classes.
EDGES = sorted({v + d for v in (12, 20, 24, 40, 48, 80, 96, 160, 320, 640, 768, 1280, 1536, 2560) for d in (-1, 0, 1)})


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distill_sizes_at_the_boundaries(dev, dtype):
    for V in EDGES:
        logits, idx, top = _record(dev, 37, V, min(V, 11), dtype, seed=V)
        _check_distill(logits, idx, top, 2.0, None, "mean", what=str(V))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [7, 21, 150, 1203, 9001])
def test_distill_writes_its_outputs_only(dev, dtype, V):
    """A gradient at an unaligned place between guard values, through the C entries: nothing around it changes."""
    from fusionsense_amd._lib import load, ptr, stream_ptr
    R, K = 45, 6
    logits, idx, top = _record(dev, R, V, K, dtype, seed=70)
    leaf = logits.clone().requires_grad_(True)
    loss = losses.topk_distill_loss(leaf, idx, top, 2.0, None, "none")
    up = _randn(dev, R, seed=71)
    want, = torch.autograd.grad(loss, [leaf], up)
    lib, dt = load(), ops.DTYPES[dtype]
    common = (64, ptr(idx), K, ops.DTYPES[torch.float32], ptr(top), K, None, 2.0)
    for off in (1, 3, 8):
        rows, stat = torch.full((R + 2,), 3.0, device=dev), torch.full((4 * R + 4,), 3.0, device=dev)
        room = torch.full((R * V + 16,), 3.0, dtype=dtype, device=dev)
        out = room[off:off + R * V]
        assert lib.fsgs_distill_fwd(R, V, K, dt, ptr(logits), V, *common, 0, rows[1:].data_ptr(), ptr(stat), None, None, 0,
                                    stream_ptr(dev)) == 0
        assert lib.fsgs_distill_bwd(R, V, K, dt, ptr(logits), V, *common, ptr(stat), None, ptr(up), 1, out.data_ptr(),
                                    stream_ptr(dev)) == 0
        assert torch.equal(rows[1:-1], loss) and torch.equal(out.reshape(R, V), want)
        assert rows[0] == 3 and rows[-1] == 3 and (stat[4 * R:] == 3).all()
        assert (room[:off] == 3).all() and (room[off + R * V:] == 3).all()
        # the scores as a slice of a wider plane: the rest of it has no gradient
        wide = torch.full((R, V + 3), float("nan"), dtype=dtype, device=dev)
        wide[:, 2:V + 2] = logits
        wide.requires_grad_(True)
        l = losses.topk_distill_loss(wide[:, 2:V + 2], idx, top, 2.0, None, "none")
        g, = torch.autograd.grad(l, [wide], up)
        assert torch.equal(l, loss) and torch.equal(g[:, 2:V + 2], want)
        assert not g[:, :2].any() and not g[:, V + 2:].any()


@pytest.mark.parametrize("tdtype", TYPES, ids=IDS)
@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_distill_types(dev, tdtype, idx_dtype):
    for dtype in TYPES:
        _check_distill(*_record(dev, 77, 40, 6, dtype, tdtype, idx_dtype, seed=4), T=1.3)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V", [19, 150, 1203, 33000])
def test_distill_rows_that_count_for_nothing(dev, dtype, V):
    """Padding of every kind, rows without entries, -inf entries, zero weights over NaN scores: exact zeros, no NaN."""
    R, K = 40, 5
    logits, idx, top = _record(dev, R, V, K, dtype, seed=31, ragged=False)
    idx[0] = -1
    idx[1] = torch.tensor([V, V + 7, -5, 2 ** 40, -2 ** 62])
    top[2] = -math.inf
    idx[3, 2:], top[3, 2:] = -1, float("nan")
    top[4, 1:] = -math.inf
    idx[5, 1] = 2 ** 32 + 3  # (its low half is a class)
    low = torch.finfo(top.dtype).min
    top[6, 2:] = low
    top[7] = low  # (all alike: uniform)
    weight = torch.ones(R, device=dev)
    weight[8] = 0.0
    logits[8] = float("nan")
    logits[0] = float("nan")
    for reduction in ops.REDUCTIONS:
        loss, grad = _check_distill(logits, idx, top, 1.0, weight, reduction, what=reduction)
        assert not grad[[0, 1, 2, 8]].any() and torch.isfinite(grad).all()
        if reduction == "none":
            assert not loss[[0, 1, 2, 8]].any()
    zero = torch.zeros(R, dtype=torch.bool, device=dev)
    for reduction in ops.REDUCTIONS:
        loss, grad = _check_distill(logits, idx, top, 1.0, zero, reduction)
        assert not loss.any() and not grad.any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distill_masked_student(dev, dtype):
    """Classes that the student rules out (-inf, the type's lowest value), and rows that are lost (NaN, all -inf)."""
    logits, idx, top = _record(dev, 12, 60, 4, dtype, seed=8, ragged=False)
    idx[:] = torch.tensor([1, 5, 9, 30])
    logits[0, 40:] = -math.inf
    logits[1, 40:] = torch.finfo(dtype).min
    logits[2] = torch.finfo(dtype).min
    loss, grad = _check_distill(logits[:3], idx[:3], top[:3], 0.5, None, "none")
    assert not grad[0, 40:].any()
    # a class the teacher wants and the student rules out: infinite loss, a gradient that pulls it back up
    logits[3, 5] = -math.inf
    leaf = logits[3:4].detach().requires_grad_(True)
    loss = losses.topk_distill_loss(leaf, idx[3:4], top[3:4], reduction="sum")
    g, = torch.autograd.grad(loss, [leaf])
    assert float(loss.detach()) == math.inf and torch.isfinite(g).all() and float(g[0, 5]) < 0
    # ... unless the teacher gives it nothing
    top[3, 1] = -math.inf
    assert torch.isfinite(losses.topk_distill_loss(logits[3:4], idx[3:4], top[3:4]))
    logits[4, 7] = float("nan")
    logits[5] = -math.inf
    top[6, 0] = float("nan")
    loss = losses.topk_distill_loss(logits[:8], idx[:8], top[:8], reduction="none")
    assert torch.isnan(loss[[4, 5, 6]]).all() and torch.isfinite(loss[[0, 1, 2, 3, 7]]).all()


def _far_scores(dev, V, K, dtype, T, seed):
    """Rows whose maximum lies anywhere in the type's range: (a) every class at one value (a mask that rules all of them out, or a
    constant), (b) a tenth of the classes around zero and the others at a mask value, (c) N(0, 2) T around an offset."""
    top = torch.finfo(dtype).max
    sizes = [s * v for v in (12.0, 345.0, 12345.0, 60000.0, 3e6, 1e9, 1e10, 1e12, 1e20, 1e30, 3e38) if v <= top for s in (1, -1)]
    g = torch.Generator().manual_seed(seed)
    rows = [torch.full((V,), v, dtype=torch.float64) for v in sizes]
    for v in sizes:
        if v < 0:
            row = torch.randn(V, generator=g, dtype=torch.float64) * 2 * T
            row[(torch.arange(V) * 7) % 10 != 0] = v
            rows.append(row)
    rows += [torch.randn(V, generator=g, dtype=torch.float64) * 2 * T + v for v in sizes]
    logits = torch.stack(rows).clamp(-top, top).to(dtype)
    R = logits.shape[0]
    # (entries among the classes around zero of (b): a ruled-out class that the teacher wants has a loss beyond fp32)
    zero = torch.arange(V)[(torch.arange(V) * 7) % 10 == 0]
    idx = zero[torch.rand(R, zero.numel(), generator=g).topk(min(K, zero.numel()), dim=1).indices]
    teacher = torch.randn(idx.shape, generator=g) * 2 * T
    return logits.to(dev), idx.to(dev), teacher.to(dev)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.5, 1.0, 30.0, 1e6])
@pytest.mark.parametrize("V", [11, 21, 150, 1203, 9001])
def test_distill_far_scores(dev, dtype, T, V):
    """Maxima over the whole range of the type, temperatures at both ends of theirs: finite, and within the bound that only
    counts differences from the row's maximum.  (A gradient goes up to T: fp16 has 65 504.)"""
    T = min(T, 1e4) if dtype == torch.float16 else T
    args = _far_scores(dev, V, 6, dtype, T, seed=91)
    for reduction in ("none", "mean"):
        loss, grad = _check_distill(*args, T, None, reduction, what=f"{reduction}")
        assert torch.isfinite(loss).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [1e-3, 1.0, 7.0])
@pytest.mark.parametrize("V", [150, 1203, 2561, 9000, 40001])
def test_distill_offset_scores(dev, dtype, T, V):
    """N(0, 2) T around a common offset over T of up to 1e6, either sign, and rows whose lanes see rising, falling and far apart
    scores: the bound counts differences from the row's maximum, not the scores themselves."""
    g = torch.Generator().manual_seed(92)
    offsets = [s * v * T for v in (0.0, 50.0, 1e3, 1e4, 1e5, 1e6) for s in (1, -1) if v * T < torch.finfo(dtype).max / 2]
    ramp = torch.linspace(-40, 0, V, dtype=torch.float64)
    rows = [torch.randn(V, generator=g, dtype=torch.float64) * 2 * T + o for o in offsets]
    rows += [r * T + o for o in offsets[-2:] for r in (ramp, ramp.flip(0), ramp[torch.randperm(V, generator=g)])]
    logits = torch.stack(rows).to(dtype).to(dev)
    R = len(rows)
    idx = torch.randint(0, V, (R, 9), generator=g)
    top = (torch.randn(R, 9, generator=g) * 2 * T + 1e3 * T).to(dev)
    for reduction in ("none", "sum"):
        _check_distill(logits, idx.to(dev), top, T, None, reduction, what=reduction)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("V,K", [(30, 8), (150, 64), (1500, 200), (33000, 70)])
def test_distill_repeated_classes(dev, dtype, V, K):
    """A class in several entries carries their sum, and two runs agree bit for bit."""
    g = torch.Generator().manual_seed(5)
    logits, _, top = _record(dev, 50, V, K, dtype, seed=6, ragged=False)
    idx = torch.randint(0, max(2, V // 10) if V < 1000 else 9, (50, K), generator=g).to(dev)
    idx[3] = 1  # (all entries the same class)
    idx[4, ::2] = -1
    l1, g1 = _check_distill(logits, idx, top, 2.0, None, "sum")
    l2, g2 = _check_distill(logits, idx, top, 2.0, None, "sum")
    assert torch.equal(l1, l2) and torch.equal(g1, g2)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_distill_layouts(dev, dtype):
    R, V, K = 60, 50, 6
    logits, idx, top = _record(dev, R, V, K, dtype, seed=13)
    weight = torch.rand(R, generator=torch.Generator().manual_seed(3)).to(dev)
    l0, g0 = _check_distill(logits, idx, top, 1.5, weight)
    wide = torch.full((R, V + 3), float("nan"), dtype=dtype, device=dev)
    wide[:, 1:V + 1] = logits
    iw = torch.full((R, K + 1), 3, dtype=idx.dtype, device=dev)
    iw[:, 1:] = idx
    tw = torch.zeros(R, K + 2, device=dev)
    tw[:, 2:] = top
    for a in ((wide[:, 1:V + 1], iw[:, 1:], tw[:, 2:], weight),
              (logits.t().contiguous().t(), idx.t().contiguous().t(), top.t().contiguous().t(), torch.stack([weight] * 2, 1)[:, 0])):
        l, g = _check_distill(*a[:3], 1.5, a[3])
        assert torch.equal(l, l0) and torch.equal(g, g0)
    l, g = _check_distill(logits.reshape(3, 20, V), idx.reshape(3, 20, K), top.reshape(3, 20, K), 1.5, weight.reshape(3, 20))
    assert torch.equal(l, l0) and torch.equal(g.reshape(R, V), g0)
    # one record for all rows
    _check_distill(logits, idx[:1].expand(R, K), top[:1].expand(R, K), 1.5, weight[:1].expand(R), "none")
    # a single row without a row axis
    _check_distill(logits[5], idx[5], top[5], 1.5, None, "none")


def test_distill_without_rows(dev):
    logits = torch.zeros(0, 9, device=dev, requires_grad=True)
    idx, top = torch.zeros(0, 2, dtype=torch.int64, device=dev), torch.zeros(0, 2, device=dev)
    for reduction in ops.REDUCTIONS:
        loss = losses.topk_distill_loss(logits, idx, top, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ())
        g, = torch.autograd.grad(loss.sum(), [logits])
        assert g.shape == (0, 9) and float(loss.sum()) == 0.0


def test_distill_refuses(dev):
    logits, idx, top = _record(dev, 4, 8, 3, torch.float32)
    for args, kw in (((logits, idx.float(), top), {}), ((logits, idx[:3], top), {}), ((logits, idx, top[:, :2]), {}),
                     ((logits, idx.cpu(), top), {}), ((logits, idx, top.double()), {}), ((logits.double(), idx, top), {}),
                     ((logits, idx, top), dict(temperature=0.0)), ((logits, idx, top), dict(temperature=float("nan"))),
                     ((logits, idx, top), dict(reduction="avg")), ((logits, idx, top), dict(weight=torch.ones(3, device=dev))),
                     ((logits, idx, top), dict(weight=torch.ones(4))), ((logits, idx[0], top[0]), {}),
                     ((logits, idx[:, :0], top[:, :0]), {}), ((logits, idx, top.clone().requires_grad_(True)), {}),
                     ((logits[:, :0], idx, top), {}),
                     ((logits, idx.repeat(1, 100), top.repeat(1, 100)), {})):
        with pytest.raises(ValueError):
            losses.topk_distill_loss(*args, **kw)


def test_distill_gradient_against_differences(dev):
    """fp32, central differences along random directions; the loss's own bound over the step, and h^2 / 6 times its third
    derivative: that of T^2 log sum exp(s / T) along d, at most 2 max|d|^3 / T per row."""
    logits, idx, top = _record(dev, 30, 40, 6, torch.float32, seed=17)
    T, h = 1.5, 2.0 ** -5
    weight = torch.rand(30, generator=torch.Generator().manual_seed(1)).to(dev)
    leaf = logits.detach().requires_grad_(True)
    g, = torch.autograd.grad(losses.topk_distill_loss(leaf, idx, top, T, weight, "sum"), [leaf])
    d = _randn(dev, 30, 40, seed=18)
    val, err = [], 0.0
    for s in (h, -h):
        moved = logits + s * d
        val.append(float(losses.topk_distill_loss(moved, idx, top, T, weight, "sum")))
        err += float(S.distill(moved, idx, top, T, weight, "sum")["loss"][1])
        err += S.U32 * abs(val[-1]) + float((2 * T * S.U32 * moved.abs().amax(1) * weight).sum())  # (the moved scores' rounding)
    third = float((2 * d.abs().amax(1) ** 3 * 4 / T * weight).sum()) * h * h / 6
    want = float((g.double() * d.double()).sum())
    assert abs((val[0] - val[1]) / (2 * h) - want) <= err / (2 * h) + third + 1e-5 * abs(want)


def test_distill_offsets_beyond_32_bits(dev):
    R, V, K, pitch = 1100, 30, 4, (1 << 21) + 1
    dtype = torch.bfloat16
    big = torch.empty(R * pitch, dtype=dtype, device=dev)
    logits0, idx, top = _record(dev, R, V, K, dtype, seed=41)
    logits = big.as_strided((R, V), (pitch, 1))
    logits.copy_(logits0)
    l0, g0 = _check_distill(logits0, idx, top)
    l, g = _check_distill(logits, idx, top)
    assert torch.equal(l, l0) and torch.equal(g, g0)
    del big, logits
    # a gradient of more than 2^31 elements: rows of one kind repeat
    V, R = 33000, (1 << 31) // 33000 + 50
    logits0, idx0, top0 = _record(dev, 50, V, K, dtype, seed=42, ragged=False)
    n = (R + 49) // 50
    leaf = logits0.repeat(n, 1)[:R].requires_grad_(True)
    loss = losses.topk_distill_loss(leaf, idx0.repeat(n, 1)[:R], top0.repeat(n, 1)[:R], reduction="none")
    g, = torch.autograd.grad(loss, [leaf], torch.ones_like(loss))
    want = S.distill(logits0, idx0, top0, reduction="none", g=torch.ones(50))
    S.check(g[:50], want["dlogits"], "first rows")
    for r0 in range(0, R, 5000):
        blk = g[r0:r0 + 5000]
        assert torch.equal(blk, g[:50].repeat(100, 1)[:blk.shape[0]]), r0
    assert torch.equal(loss, loss[:50].repeat(n)[:R])


# ---- both together --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(dev, grad):
    """A tangent is refused, never lost."""
    from torch.autograd import forward_ad
    x, w, b, r, _ = _layer(dev, 6, 8, 5, torch.float32)
    logits, idx, top = _record(dev, 6, 8, 3, torch.float32, ragged=False)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        for i in range(4):
            args = [x, w, b, "gelu", r]
            i += i == 3
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                ops.linear_act(*args)
        with pytest.raises(NotImplementedError):
            losses.topk_distill_loss(forward_ad.make_dual(logits, torch.ones_like(logits)), idx, top)
        with pytest.raises(NotImplementedError):
            losses.topk_distill_loss(logits, idx, forward_ad.make_dual(top, torch.ones_like(top)))
        ops.linear_act(x, w, b, "gelu", r), losses.topk_distill_loss(logits, idx, top)


def _step(head, feats, idx, top, weight):
    logits = head(feats)
    loss = losses.topk_distill_loss(logits, idx, top, 2.0, weight)
    return loss, torch.autograd.grad(loss, [feats] + list(head.parameters()))


def test_head_and_loss_against_64_bits(dev):
    """fp32 head of three layers and the loss on it, all gradients, against torch's autograd in fp64.  The tolerance follows the
    values: a layer's outputs are off by (K + 2) U32 of its terms' magnitudes, which the next layer's gradients carry on; with
    3 layers of width <= 64 that is below 3 * 66 U32 * (amplification, at most 8 for weights of bound 1 / sqrt K and these
    activations) of a tensor's largest gradient: 1e-4 of it."""
    R, V, K = 700, 150, 8
    head = SemanticHead(32, V, hidden=64, blocks=1, device=dev, generator=torch.Generator().manual_seed(0))
    feats = _randn(dev, R, 32, seed=1).requires_grad_(True)
    _, idx, top = _record(dev, R, V, K, torch.float32, torch.float16, torch.int32, seed=2)
    weight = torch.rand(R, generator=torch.Generator().manual_seed(4)).to(dev)
    loss, grads = _step(head, feats, idx, top, weight)
    leaves = [t.detach().cpu().double().requires_grad_(True) for t in [feats] + list(head.parameters())]
    f, (w0, w1, w2, b0, b1, b2) = leaves[0], leaves[1:]
    h0 = S.act(f @ w0.t() + b0, "gelu")
    h1 = S.act(h0 @ w1.t() + b1, "gelu") + h0
    s = h1 @ w2.t() + b2
    i, t = idx.cpu().long(), top.cpu().double()
    pad = i < 0
    alive = ~pad.all(1)
    lp = torch.log_softmax((t / 2.0).masked_fill(pad, -1e30), 1)
    p = lp.exp().masked_fill(pad, 0.0)
    lq = torch.gather(torch.log_softmax(s / 2.0, 1), 1, i.clamp(min=0))
    rows = 4.0 * (p * (lp - lq)).masked_fill(pad, 0.0).sum(1)
    w = weight.cpu().double() * alive
    want = (rows * w).sum() / w.sum()
    assert abs(float(loss) - float(want)) < 1e-5 * abs(float(want))
    for got, ref in zip(grads, torch.autograd.grad(want, leaves)):
        assert (got.cpu().double() - ref).abs().max() <= 1e-4 * ref.abs().max()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_head_and_loss_captured_and_on_another_stream(dev, dtype):
    """Two captured training steps, replayed in turn with eager work between, and a step on a side stream: the eager step's
    bits each time (no state is shared between them)."""
    R, V, K = 1111, 150, 8

    def make(seed):
        head = SemanticHead(32, V, hidden=64, dtype=dtype, device=dev, generator=torch.Generator().manual_seed(seed))
        feats = _randn(dev, R, 32, seed=seed, dtype=dtype).requires_grad_(True)
        _, idx, top = _record(dev, R, V, K, torch.float32, torch.float16, seed=seed)
        return head, feats, idx, top, torch.rand(R, generator=torch.Generator().manual_seed(seed)).to(dev)
    sets = [make(1), make(2)]
    side = torch.cuda.Stream()
    graphs, outs, want = [], [], []
    for a in sets:
        loss, grads = _step(*a)
        want.append([loss.detach().clone()] + [g.clone() for g in grads])
        del loss, grads
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            loss, grads = _step(*a)
            got = [loss.detach()] + list(grads)
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want[-1]))
        del loss, grads, got
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, grads = _step(*a)
            out = [loss.detach()] + list(grads)
        del loss, grads
        graphs.append(g)
        outs.append(out)
    for rep in range(3):
        for i in (0, 1, 1, 0):
            for t in outs[i]:
                t.fill_(7.0)
            graphs[i].replay()
            (sets[i][1].detach() * 2).sum().item()
            assert all(torch.equal(x, y) for x, y in zip(outs[i], want[i])), (rep, i)
    # new inputs in the captured buffers: the replay follows them
    with torch.no_grad():
        sets[0][1].mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in outs[0]]
    loss, grads = _step(*sets[0])
    assert all(torch.equal(x, y) for x, y in zip(got, [loss.detach()] + list(grads)))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("R", [5, 700])
def test_wide_head_and_loss_captured_and_on_two_streams(dev, dtype, act, R):
    """A head too wide for the one-pass backward, few points and many: a captured step replayed with eager work between, and two
    steps at once on two streams, give the eager step's bits."""
    head = SemanticHead(40, 2700, hidden=600, blocks=1, act=act, dtype=dtype, device=dev,
                        generator=torch.Generator().manual_seed(1))

    def data(seed):
        feats = _randn(dev, R, 40, seed=seed, dtype=dtype).requires_grad_(True)
        _, idx, top = _record(dev, R, 2700, 8, torch.float32, torch.float16, seed=seed)
        return feats, idx, top, torch.rand(R, generator=torch.Generator().manual_seed(seed)).to(dev)
    sets, want = [data(1), data(2)], []
    for a in sets:
        loss, grads = _step(head, *a)
        want.append([loss.detach().clone()] + [g.clone() for g in grads])
        del loss, grads
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                loss, grads = _step(head, *sets[i])
                got[i] = [loss.detach()] + list(grads)
                del loss, grads
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(x, y) for x, y in zip(got[i], want[i]))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = _step(head, *sets[0])
        out = [loss.detach()] + list(grads)
    del loss, grads
    for _ in range(3):
        for t in out:
            t.fill_(7.0)
        graph.replay()
        (sets[0][0].detach() * 2).sum().item()
        assert all(torch.equal(x, y) for x, y in zip(out, want[0]))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_head_and_loss_with_saved_tensors_kept_on_the_host(dev, dtype):
    """What the backward needs may come back in other storage and with other strides: the same bits."""
    head = SemanticHead(32, 150, hidden=64, dtype=dtype, device=dev, generator=torch.Generator().manual_seed(0))
    wide = _randn(dev, 333, 35, seed=1, dtype=dtype)
    _, idx, top = _record(dev, 333, 150, 8, torch.float32, seed=2)
    out = []
    for hooks in (False, True):
        feats = wide.clone().requires_grad_(True)
        with torch.autograd.graph.save_on_cpu(pin_memory=False) if hooks else torch.enable_grad():
            loss = losses.topk_distill_loss(head(feats[:, 1:33]), idx, top, 2.0)
        out.append(torch.autograd.grad(loss, [feats] + list(head.parameters())))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_semantics_through_the_renderer(dev):
    """render_fusionsense with a head: the plane is the features' composite, the scores are the head's, the loss's gradient
    reaches the feature rows and the head and stops at the geometry; images are what they are without the head."""
    params, cam = scenes.cube_scene(1000, seed=0)
    p = {k: v.to(dev).requires_grad_(True) for k, v in params.items()}
    p["semantics"] = _randn(dev, 1000, 10, seed=1).requires_grad_(True)
    head = SemanticHead(10, 21, hidden=16, device=dev, generator=torch.Generator().manual_seed(0))
    out = render_fusionsense(p, cam, semantic_head=head)
    plain = render_fusionsense({k: v for k, v in p.items() if k != "semantics"}, cam)
    H, W = cam.height, cam.width
    assert out["semantic_features"].shape == (H, W, 10) and out["semantic_logits"].shape == (H, W, 21)
    for k in ("rgb", "depth", "normal", "accumulation"):
        assert torch.equal(out[k], plain[k]), k
    assert "semantic_logits" not in plain
    # features of ones composite to the accumulation
    ones = dict(p, semantics=torch.ones(1000, 10, device=dev))
    f = render_fusionsense(ones, cam, semantic_head=head)["semantic_features"]
    assert (f - out["accumulation"]).abs().max() < 1e-5
    _, idx, top = _record(dev, H * W, 21, 4, torch.float32, seed=3)
    loss = losses.topk_distill_loss(out["semantic_logits"], idx.reshape(H, W, 4), top.reshape(H, W, 4), 1.0,
                                    (out["accumulation"].detach()[..., 0] > 0.5))
    loss.backward()
    assert p["semantics"].grad.abs().sum() > 0 and all(q.grad.abs().sum() > 0 for q in head.parameters())
    assert all(p[k].grad is None for k in params)
    with pytest.raises(ValueError, match="semantics"):
        render_fusionsense({k: v for k, v in p.items() if k != "semantics"}, cam, semantic_head=head)
    # a crop that leaves nothing: scores of a zero plane
    from fusionsense_amd.crop import OrientedBox
    box = OrientedBox(torch.eye(3), torch.full((3,), 100.0), torch.ones(3))
    with torch.no_grad():
        e = render_fusionsense(p, cam, semantic_head=head, crop_box=box, training=False)
        assert not e["semantic_features"].any()
        assert torch.equal(e["semantic_logits"], head(torch.zeros(H, W, 10, device=dev)))


def test_semantic_features_train_through_the_renderer(dev):
    """The feature rows' gradient against differences of the whole chain (render, head, loss) along one direction, step 2^-7:
    the scores are linear in the rows up to the head (|gelu'''| <= 2), so the quotient's cubic term is below 1e-3 of the
    gradient here, and fp32's 1e-6 of the loss over the step 1e-4 of it."""
    params, cam = scenes.cube_scene(300, seed=2)
    p = {k: v.to(dev) for k, v in params.items()}
    feats = _randn(dev, 300, 8, seed=5)
    head = SemanticHead(8, 12, hidden=16, device=dev, generator=torch.Generator().manual_seed(3))
    H, W = cam.height, cam.width
    _, idx, top = _record(dev, H * W, 12, 3, torch.float32, seed=6, ragged=False)

    def value(f):
        lg = render_fusionsense(dict(p, semantics=f), cam, semantic_head=head)["semantic_logits"]
        return losses.topk_distill_loss(lg, idx.reshape(H, W, 3), top.reshape(H, W, 3))
    leaf = feats.clone().requires_grad_(True)
    g, = torch.autograd.grad(value(leaf), [leaf])
    d = g / g.abs().max()
    h = 2.0 ** -7
    with torch.no_grad():
        q = (float(value(feats + h * d)) - float(value(feats - h * d))) / (2 * h)
    want = float((g.double() * d.double()).sum())
    assert abs(q - want) <= 0.01 * abs(want) + 2 * S.U32 * 64 * float(value(feats).detach()) / (2 * h)
