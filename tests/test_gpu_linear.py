"""GPU: the products with their epilogues (fused_linear_*), the routed experts' ragged products
(grouped_linear_*) and their plan (moe_group_rows) against the formulas in 64 bits.

Bounds, elementwise. u = 2^-24 (half a step of fp32), h = half a step of the output's type
(2^-8 bf16, u fp32), S = |x| |w| + |bias|.
  pre: a sum of n products in fp32 is off by at most n u S in any order, rounding by h |pre|.
  y:   that error d times the activation's steepest slope (1.13), its evaluation within 16 u
       (|pre| + 1), rounding h |y|. SwiGLU: the product rule over both halves.
  dpre = act'(pre) dy in fp32 within 2^-18 |dy| (slopes up to 1.13 with exponents' arguments
       up to 100, each rounded), then rounded to the type: h |dpre|. SwiGLU: times |u| + |g|.
  dx, dw, db: the rounding of dpre through the sum, n u of the sum of magnitudes, rounding h.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "swiglu")


@pytest.fixture(scope="module")
def pc():
    import pulsar_cuda

    return pulsar_cuda


def half(dt):
    return torch.finfo(dt).eps / 2


def rand(*shape, seed, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt).cuda()


def act64(act, p):
    if act == "none":
        return p
    if act == "relu":
        return p.clamp_min(0)
    if act == "silu":
        return p * torch.sigmoid(p)
    if act == "gelu":
        return p * torch.special.ndtr(p)
    if act == "gelu_tanh":
        return 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)))
    if act == "sigmoid":
        return torch.sigmoid(p)
    g, u = p.chunk(2, -1)
    return g * torch.sigmoid(g) * u


def check(got, want, tol, what):
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    g = got.double()
    bad = ~((g - want).abs() <= tol)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst error "
        f"{(g - want).abs().max().item():.3e} where the bound is {tol.min().item():.3e} or more")


def check_forward(got_y, got_pre, x, w, bias, act, dt, res=None, what=""):
    """x [M, I], w [I, O] of one group."""
    x, w = x.double(), w.double()
    n = x.shape[1] + 2
    b = 0 if bias is None else bias.double()
    pre = x @ w + b
    S = x.abs() @ w.abs() + (0 if bias is None else b.abs())
    d = n * U * S
    y = act64(act, pre)
    if act == "swiglu":
        g, u = pre.chunk(2, -1)
        dg, du = d.chunk(2, -1)
        ty = 1.13 * dg * u.abs() + g.abs() * du + dg * du + 16 * U * (g.abs() + 1) * (u.abs() + 1)
    else:
        ty = 1.13 * d + 16 * U * (pre.abs() + 1)
    if res is not None:
        y = y + res.double()
        ty = ty + U * y.abs()
    check(got_y, y, half(dt) * (y.abs() + ty) + ty, what + " y")
    if got_pre is not None:
        check(got_pre, pre, half(dt) * (pre.abs() + d) + d, what + " pre")


def dpre64(act, pre, dy):
    """act'(pre) dy and the bound of its error before rounding."""
    leaf = pre.double().requires_grad_()
    (d,) = torch.autograd.grad(act64(act, leaf), leaf, dy.double())
    if act == "none":
        return d, torch.zeros_like(d)
    if act == "swiglu":
        g, u = pre.double().abs().chunk(2, -1)
        e = 2.0 ** -18 * dy.double().abs()
        return d, torch.cat([e * u, e * g], -1)
    return d, 2.0 ** -18 * dy.double().abs()


def check_backward(dx, dw, db, dy, x, w, pre, act, dt, what=""):
    """One group: x [M, I], w and dw [I, O]."""
    d, e = dpre64(act, pre, dy)
    h = half(dt) if act != "none" else 0.0
    ed = e + h * (d.abs() + e)  # error of the rounded dpre
    x, w = x.double(), w.double()
    for got, want, mag, n, name in (
            (dx, d @ w.t(), (d.abs() + ed) @ w.t().abs(), d.shape[1], "dx"),
            (dw, x.t() @ d, x.t().abs() @ (d.abs() + ed), d.shape[0], "dw"),
            (db, d.sum(0), (d.abs() + ed).sum(0), d.shape[0], "db")):
        if got is None:
            continue
        through = {"dx": lambda: ed @ w.t().abs(), "dw": lambda: x.t().abs() @ ed,
                   "db": lambda: ed.sum(0)}[name]()
        t = through + (n + 2) * U * mag
        check(got, want, half(dt) * (want.abs() + t) + t, f"{what} {name}")


# --------------------------------------------------------------------------------------
# moe_group_rows
# --------------------------------------------------------------------------------------

def group_ref(idx, E):
    N, K = idx.shape
    flat = idx.reshape(-1)
    valid = (flat >= 0) & (flat < E)
    order = np.argsort(np.where(valid, flat, E), kind="stable")
    n = int(valid.sum())
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[valid], minlength=E))])
    rows = np.full(N * K, -1)
    rows[:n] = order[:n] // K
    slots = np.full(N * K, -1)
    slots[order[:n]] = np.arange(n)
    return offsets, rows, slots.reshape(N, K)


@pytest.mark.parametrize("N,K,E", [
    (0, 4, 16), (1, 1, 1), (1, 4, 16), (3, 2, 5), (17, 3, 7), (64, 1, 2), (1024, 4, 16),
    (1025, 4, 16), (683, 6, 63), (4097, 1, 64), (2048, 8, 65), (16384, 4, 16), (9001, 8, 1000),
    (5000, 2, 1024), (90000, 3, 33), (300000, 1, 1)])
@pytest.mark.parametrize("padded", [False, True])
def test_group_rows(pc, N, K, E, padded):
    rng = np.random.default_rng(N + E)
    idx = rng.integers(0, max(1, E - E // 4), size=(N, K))  # the last experts stay empty
    if padded and N:
        idx[rng.random((N, K)) < 0.2] = rng.choice([-1, E, E + 7, -2 ** 40, 2 ** 40])
    got = pc.moe_group_rows(torch.from_numpy(idx).cuda(), E)
    for g, w, name in zip(got, group_ref(idx, E), ("offsets", "rows", "slots")):
        assert g.dtype == torch.int32
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)


# --------------------------------------------------------------------------------------
# fused_linear
# --------------------------------------------------------------------------------------

SHAPES = [(1, 1, 2), (1, 64, 64), (1, 1024, 1024), (3, 8, 16), (16, 1024, 1040), (17, 33, 66),
          (65, 72, 136), (129, 100, 130), (130, 1000, 776), (300, 1023, 778), (520, 64, 2048)]


def _off(t):
    """The same values at a pointer one element past a 16-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:].copy_(t.reshape(-1))
    return buf[1:].view(t.shape)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,I,O", SHAPES)
@pytest.mark.parametrize("order", ["oi", "io"])
def test_linear_shapes(pc, M, I, O, order, dtype):
    dt = DT[dtype]
    x, dy = rand(M, I, seed=1, dt=dt), rand(M, O, seed=4, dt=dt)
    w = rand(O, I, seed=2, dt=dt, scale=I ** -0.5)
    if order == "io":
        w = w.t().contiguous().t()
    b = rand(O, seed=3, dt=dt)
    for act in ("none", "silu", "swiglu"):
        d = dy[:, : O // 2].contiguous() if act == "swiglu" else dy
        for shift in (lambda t: t, _off):
            xx = shift(x)
            y, pre = pc.fused_linear_forward(xx, w, b, act, save_pre=True)
            check_forward(y, pre, x, w.t(), b, act, dt, what=act)
            dx, dw, db = pc.fused_linear_backward(shift(d), xx, w, shift(pre), act, bias=True)
            assert dw.stride() == w.stride() or 1 in w.shape
            check_backward(dx, dw.t(), db, d, x, w.t(), pre, act, dt, what=act)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(pc, act, dtype):
    """Every activation, residual and bias type, with values far out on both sides."""
    dt = DT[dtype]
    M, I, O = 70, 64, 96
    x = rand(2, M // 2, I, seed=5, dt=dt, scale=4.0)
    w = rand(O, I, seed=6, dt=dt)
    x[0, 0] *= 100
    cols = O // 2 if act == "swiglu" else O
    res = rand(2, M // 2, cols, seed=7, dt=dt)
    for bias in (None, rand(O, seed=8, dt=dt), rand(O, seed=9, dt=torch.float32)):
        y, pre = pc.fused_linear_forward(x, w, bias, act, residual=res, save_pre=True)
        assert y.shape == (2, M // 2, cols)
        check_forward(y.view(M, -1), pre.view(M, -1), x.view(M, I), w.t(), bias, act, dt,
                      res=res.view(M, -1), what=act)
        assert torch.equal(y, pc.fused_linear_forward(x, w, bias, act, residual=res))
    dy = rand(2, M // 2, cols, seed=10, dt=dt)
    dx, dw, db = pc.fused_linear_backward(dy, x, w, pre, act, bias=False)
    assert db is None and dx.shape == x.shape
    check_backward(dx.view(M, I), dw.t(), None, dy.view(M, -1), x.view(M, I), w.t(),
                   pre.view(M, -1), act, dt, what=act)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh", "sigmoid"])
def test_activation_gradient_at_the_ends(pc, act):
    """Slopes at +-infinity and the largest numbers are their limits; NaN stays NaN."""
    big = torch.tensor([float("inf"), 3e38, 1e20, 200.0, -200.0, -1e20, -3e38, -float("inf"),
                        float("nan")], device="cuda").view(-1, 1)
    M = big.numel()
    x, w, dy = torch.zeros(M, 1, device="cuda"), torch.ones(1, 1, device="cuda"), torch.ones_like(big)
    dx, _, _ = pc.fused_linear_backward(dy, x, w, big, act)
    up = 0.0 if act == "sigmoid" else 1.0
    assert dx[:4].flatten().tolist() == [up] * 4
    assert dx[4:8].flatten().tolist() == [0.0] * 4
    assert bool(dx[8].isnan())


@pytest.mark.parametrize("dtype", list(DT))
def test_swiglu_gradient_of_large_dy(pc, dtype):
    """dy g and dy u pass fp32's range where the gradients, dy silu(g) and dy u silu'(g), are far
    inside it. One row: the bias gradient is dpre itself."""
    dt = DT[dtype]
    g = torch.tensor([-200.0, -60.0, -60.0, -200.0])
    u = torch.tensor([1000.0, 1000.0, -1000.0, 0.0])
    pre = torch.cat([g, u])[None].to(dt).cuda()
    dy = torch.tensor([[1e37, 1e37, -1e37, 3e38]]).to(dt).cuda()
    x, w = rand(1, 8, seed=1, dt=dt), torch.zeros(8, 8, dtype=dt, device="cuda")
    dx, dw, db = pc.fused_linear_backward(dy, x, w, pre, "swiglu", True)
    want, e = dpre64("swiglu", pre, dy)
    # e^g's argument is rounded to |g| u relative, more than e's share of dy u for |g| = 60; and
    # what fp32's exponent range cannot hold (e^-200 is 0) is below 2^-126 of the other factors
    e = 1e-4 * want.abs() + 2.0 ** -100 * (dy.double().abs().repeat(1, 2))
    check(db[None], want, half(dt) * (want.abs() + e) + e, "db")
    assert not dx.any() and torch.isfinite(dw).all()


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_strided_operands(pc, dtype):
    """x, residual and weight as column slices of wider buffers, aligned and not; what lies
    beside them (NaN) is not read into any result."""
    dt = DT[dtype]
    M, I, O = 150, 72, 104
    for off in (0, 8, 3):
        def cut(r, c, seed, o=off):
            buf = torch.full((r, c + 16), float("nan"), dtype=dt, device="cuda")
            buf[:, o:o + c] = rand(r, c, seed=seed, dt=dt, scale=0.3)
            return buf[:, o:o + c]
        x, w, wt, res = cut(M, I, 1), cut(O, I, 2), cut(I, O, 3).t(), cut(M, O, 4)
        for ww in (w, wt):
            y, pre = pc.fused_linear_forward(x, ww, None, "gelu", residual=res, save_pre=True)
            check_forward(y, pre, x, ww.t(), None, "gelu", dt, res=res)
            dy = rand(M, O, seed=5, dt=dt)
            dx, dw, db = pc.fused_linear_backward(dy, x, ww, pre, "gelu", bias=True)
            check_backward(dx, dw.t(), db, dy, x, ww.t(), pre, "gelu", dt)


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_no_rows(pc, dtype):
    dt = DT[dtype]
    x, w = torch.empty(0, 64, dtype=dt, device="cuda"), rand(32, 64, seed=1, dt=dt)
    y, pre = pc.fused_linear_forward(x, w, None, "swiglu", save_pre=True)
    assert y.shape == (0, 16) and pre.shape == (0, 32)
    dx, dw, db = pc.fused_linear_backward(y, x, w, pre, "swiglu", bias=True)
    assert dx.shape == (0, 64) and not dw.any() and not db.any() and dw.shape == w.shape


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_split_sums(pc, dtype):
    """Long sums of a small weight gradient, split over workgroups: same bits on every call."""
    dt = DT[dtype]
    M, I, O = 9001, 72, 40
    x, w, dy = rand(M, I, seed=1, dt=dt), rand(O, I, seed=2, dt=dt), rand(M, O, seed=3, dt=dt)
    for ww in (w, w.t().contiguous().t()):
        a = pc.fused_linear_backward(dy, x, ww, bias=True)
        check_backward(a[0], a[1].t(), a[2], dy, x, ww.t(), dy, "none", dt)
        for p, q in zip(a, pc.fused_linear_backward(dy, x, ww, bias=True)):
            assert torch.equal(p, q)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_linear_gradient_by_differences(pc, act):
    """fp32 gradients against central differences of the kernel's own forward: step 2^-6, sums of
    about 100 terms, so the difference quotient is good to about 1e-3 of the gradient's size."""
    x, w = rand(7, 24, seed=1, dt=torch.float32), rand(20, 24, seed=2, dt=torch.float32, scale=0.2)
    y, pre = pc.fused_linear_forward(x, w, None, act, save_pre=True)
    dy = rand(*y.shape, seed=3, dt=torch.float32)
    dx, dw, _ = pc.fused_linear_backward(dy, x, w, pre, act)
    f = lambda xx, ww: float((pc.fused_linear_forward(xx, ww, None, act).double() * dy.double()).sum())
    s = 2.0 ** -6
    for t, g, other in ((x, dx, lambda v: f(v, w)), (w, dw, lambda v: f(x, v))):
        for k in (0, 5, t.numel() // 2, t.numel() - 1):
            e = torch.zeros_like(t)
            e.view(-1)[k] = s
            num = (other(t + e) - other(t - e)) / (2 * s)
            assert abs(num - float(g.reshape(-1)[k])) <= 2e-3 * float(g.abs().max())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("M,I,O", [(4096, 64, 2048), (20000, 72, 264), (16384, 1024, 1024),
                                   (36001, 1024, 1000), (38500, 1024, 1024)])
def test_linear_many_tiles(pc, M, I, O, dtype):
    """Launches of many tiles of every shape: whole rounds of the chip, and last tiles that two or
    four workgroups share (1024 wide); residual, kept values, both orders."""
    dt = DT[dtype]
    x, res = rand(M, I, seed=1, dt=dt), rand(M, O, seed=2, dt=dt)
    dy = rand(M, O, seed=3, dt=dt)
    w, b = rand(O, I, seed=4, dt=dt, scale=I ** -0.5), rand(O, seed=5, dt=dt)
    for ww in (w, w.t().contiguous().t()):
        for act in ("none", "gelu", "silu"):
            y, pre = pc.fused_linear_forward(x, ww, b, act, residual=res, save_pre=True)
            check_forward(y, pre, x, ww.t(), b, act, dt, res=res, what=act)
        check_forward(pc.fused_linear_forward(x, ww), None, x, ww.t(), None, "none", dt)
        check_forward(pc.fused_linear_forward(x, ww, b, "swiglu"), None, x, ww.t(), b, "swiglu", dt)
        dx, dw, db = pc.fused_linear_backward(dy, x, ww, pre, "silu", bias=True)
        check_backward(dx, dw.t(), db, dy, x, ww.t(), pre, "silu", dt)


@pytest.mark.parametrize("M,I,O", [(5, 64, 48), (300, 200, 264), (700, 1024, 520)])
def test_linear_fp32_infinities(pc, M, I, O):
    """fp32 sums with infinities, NaN and values beyond bf16's range are those of fp32: the same
    finite results, infinities of the same sign and NaNs as torch's products."""
    x, w = rand(M, I, seed=1, dt=torch.float32), rand(O, I, seed=2, dt=torch.float32)
    x[1, 3], x[2, 5], x[3, 7], x[4, 1] = float("inf"), -float("inf"), float("nan"), 3.4e38
    w[:, 1] *= 0.25
    w[7, 9] = 3.4e38
    x[0, 9] = 0.0
    dy = rand(M, O, seed=3, dt=torch.float32)
    y = pc.fused_linear_forward(x, w)
    dx, dw, db = pc.fused_linear_backward(dy, x, w, bias=True)
    ref = x.double() @ w.double().t()
    for got, a, b in ((y, x.double(), w.double().t()), (dx, dy.double(), w.double()),
                      (dw, dy.double().t(), x.double())):
        want = a @ b
        n = a.shape[1] + 2
        # a finite product past fp32's range is an infinity in fp32 and not in 64 bits: with one of
        # the other sign in the sum it gives NaN (inf - inf), without one an infinity. Sums that
        # hold such a product have no 64-bit counterpart. Magnitudes: the sum of the finite
        # factors' products bounds each of them.
        fa, fb = (torch.where(t.isfinite(), t, 0.0) for t in (a, b))
        S = fa.abs() @ fb.abs()
        there = S < 3.4e38
        fin = torch.isfinite(want) & there
        assert bool(((got.double() - want)[fin].abs() <= n * U * S[fin] + U * want[fin].abs()).all())
        assert torch.equal(got.isnan() & there, want.isnan() & there)
        inf = torch.isinf(want) & there
        assert torch.equal(got[inf].double(), want[inf])
        assert bool(there.any())
    assert ref.isnan().any() and torch.isinf(ref).any()


# --------------------------------------------------------------------------------------
# grouped_linear
# --------------------------------------------------------------------------------------

COUNTS = [[5], [0, 3, 0], [1] * 7, [64, 0, 65, 1, 130], [0, 0], [300, 17, 0, 128, 2, 63],
          [3, 0] * 40 + [129], [1] * 130, [2] * 63, [3] * 64, [4000, 100, 0, 5200, 257]]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("counts", COUNTS, ids=[str(i) for i in range(len(COUNTS))])
@pytest.mark.parametrize("I,O,order,gather", [
    (64, 96, "io", True), (72, 40, "oi", True), (33, 50, "io", False), (33, 50, "oi", True),
    (1, 2, "io", False), (256, 264, "io", False), (136, 130, "oi", False)])
def test_grouped(pc, counts, I, O, order, gather, dtype):
    dt = DT[dtype]
    E, M = len(counts), sum(counts)
    tail = 9  # rows of no group
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()
    w = rand(E, I, O, seed=1, dt=dt, scale=I ** -0.5)
    for e, c in enumerate(counts):
        if c == 0:
            w[e] = float("nan")  # the weights of a group without rows meet nothing
    if order == "oi":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    if gather:
        R = M // 2 + 3
        rows = torch.randint(0, R - 1, (M + tail,), generator=torch.Generator().manual_seed(3))
        rows[M:] = torch.randint(-5, R + 5, (tail,), generator=torch.Generator().manual_seed(4))
        rows = rows.to(torch.int32).cuda()
        x = rand(R, I, seed=2, dt=dt)
        x[R - 1] = float("nan")  # named by rows of no group only
        xs = x[rows[:M].long()]
    else:
        rows, x = None, rand(M + tail, I, seed=2, dt=dt)
        x[M:] = float("nan")
        xs = x[:M]
    b = rand(E, O, seed=5, dt=dt)
    for act in ("none", "swiglu"):
        y, pre = pc.grouped_linear_forward(x, w, offsets, rows, b, act, save_pre=True)
        assert not y[M:].any() and not pre[M:].any()
        dy = rand(M + tail, y.shape[1], seed=6, dt=dt)
        dy[M:] = float("nan")
        dx, dw, db = pc.grouped_linear_backward(dy, x, w, offsets, rows, pre, act, bias=True)
        assert not dx[M:].any() and dx.shape == (M + tail, I)
        assert dw.stride() == w.stride() or 1 in (I, O)
        s = 0
        for e, c in enumerate(counts):
            if c == 0:
                assert not dw[e].any() and not db[e].any()
                continue
            q = slice(s, s + c)
            s += c
            check_forward(y[q], pre[q], xs[q], w[e], b[e], act, dt, what=f"group {e}")
            check_backward(dx[q], dw[e], db[e], dy[q], xs[q], w[e], pre[q], act, dt,
                           what=f"group {e}")
        y2 = pc.grouped_linear_forward(x, w, offsets, rows, b, act)
        assert torch.equal(y, y2)
        for p, r in zip((dx, dw, db), pc.grouped_linear_backward(dy, x, w, offsets, rows, pre, act,
                                                                 bias=True)):
            assert torch.equal(p, r)


@pytest.mark.parametrize("order", ["io", "oi"])
def test_grouped_many_rows(pc, order):
    """50,000 rows in uneven groups: the largest tiles, the last of them shared, group ends inside
    shared tiles, gathered rows."""
    dt, I, O = torch.bfloat16, 1024, 1024
    counts = [20011, 0, 7, 9000, 256, 12345, 1, 8421]
    M, R = sum(counts), 9000
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()
    rows = torch.randint(0, R, (M + 40,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    x, w = rand(R, I, seed=2, dt=dt), rand(len(counts), I, O, seed=3, dt=dt, scale=I ** -0.5)
    if order == "oi":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    for act in ("none", "swiglu"):
        y, pre = pc.grouped_linear_forward(x, w, offsets, rows, None, act, save_pre=True)
        dy = rand(*y.shape, seed=4, dt=dt)
        dx, dw, db = pc.grouped_linear_backward(dy, x, w, offsets, rows, pre, act, bias=True)
        assert not y[M:].any() and not pre[M:].any() and not dx[M:].any()
        s = 0
        for e, c in enumerate(counts):
            q, s = slice(s, s + c), s + c
            if c == 0:
                assert not dw[e].any()
                continue
            xs = x[rows[q].long()]
            check_forward(y[q], pre[q], xs, w[e], None, act, dt, what=f"group {e}")
            check_backward(dx[q], dw[e], db[e], dy[q], xs, w[e], pre[q], act, dt, what=f"group {e}")


@pytest.mark.parametrize("dtype", list(DT))
def test_grouped_index_outside_x(pc, dtype):
    """A row an index outside x names is a row of zeros, in the product and in the gradient."""
    dt = DT[dtype]
    x, w = rand(6, 64, seed=1, dt=dt), rand(2, 64, 32, seed=2, dt=dt)
    rows = torch.tensor([0, -1, 5, 6, 2 ** 31 - 1, 3, -2 ** 31], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 4, 7], dtype=torch.int32).cuda()
    xs = torch.zeros(7, 64, dtype=dt, device="cuda")
    for i, r in enumerate(rows.tolist()):
        if 0 <= r < 6:
            xs[i] = x[r]
    dy = rand(7, 32, seed=3, dt=dt)
    b = rand(2, 32, seed=4, dt=dt)
    assert torch.equal(pc.grouped_linear_forward(x, w, offsets, rows, b),
                       pc.grouped_linear_forward(xs, w, offsets, None, b))
    for p, q in zip(pc.grouped_linear_backward(dy, x, w, offsets, rows, bias=True),
                    pc.grouped_linear_backward(dy, xs, w, offsets, None, bias=True)):
        assert torch.equal(p, q)
    # x without rows
    assert not pc.grouped_linear_forward(x[:0], w, offsets, rows).any()


@pytest.mark.parametrize("dtype", list(DT))
def test_grouped_odd_offsets_stay_in_bounds(pc, dtype):
    """Offsets that fall, start past 0 or pass the rows address nothing outside the operands (the
    kernels hold them to [0, M]); groups that are in order keep their results."""
    dt = DT[dtype]
    x, w, dy = rand(40, 64, seed=1, dt=dt), rand(3, 64, 32, seed=2, dt=dt), rand(40, 32, seed=3, dt=dt)
    for off in ([5, 10, 20, 40], [0, 30, 10, 40], [-9, 7, 90, 2 ** 31 - 1]):
        o = torch.tensor(off, dtype=torch.int32).cuda()
        y = pc.grouped_linear_forward(x, w, o)
        pc.grouped_linear_backward(dy, x, w, o, bias=True)
        a, b = max(off[0], 0), off[1]
        check_forward(y[a:min(b, 10)], None, x[a:min(b, 10)], w[0], None, "none", dt)
    torch.cuda.synchronize()


def _moe(pc, x, idx, wt, w_gu, w_down, shared, E):
    off, rows, slots = pc.moe_group_rows(idx, E)
    act, gu = pc.grouped_linear_forward(x, w_gu, off, rows, activation="swiglu", save_pre=True)
    eo = pc.grouped_linear_forward(act, w_down, off)
    one = torch.zeros_like(idx)
    y = pc.moe_combine_forward(eo[None], one, wt, slots, shared)
    return y, (off, rows, slots, act, gu, eo, one)


def _moe_backward(pc, dy, x, wt, w_gu, w_down, saved):
    off, rows, slots, act, gu, eo, one = saved
    d_eo, d_wt = pc.moe_combine_backward(dy, eo[None], one, wt, slots)
    d_act, d_down, _ = pc.grouped_linear_backward(d_eo[0], act, w_down, off)
    d_x, d_gu, _ = pc.grouped_linear_backward(d_act, x, w_gu, off, rows, gu, "swiglu")
    return pc.moe_dispatch_backward(d_x[None], one, slots, *x.shape), d_gu, d_down, d_wt


@pytest.mark.parametrize("N,D,F,E,K", [(1, 64, 32, 4, 2), (37, 128, 64, 16, 4), (600, 256, 136, 8, 3)])
def test_experts_without_capacity(pc, N, D, F, E, K):
    """Plan, gate/up product, down product and combine, forward and backward, against the MoE
    formula in 64 bits. Each bf16 op rounds once (h = 2^-8): three roundings in a row on the
    forward path, five on the longest gradient path, random and independent; the bound is
    that many h of the result's largest magnitude. fp32: 1e-5 of it (sums of up to 600
    products of 2^-24)."""
    for dtype, fwd, bwd in (("fp32", 1e-5, 1e-5), ("bf16", 3 * 2.0 ** -8, 5 * 2.0 ** -8)):
        dt = DT[dtype]
        x, dy = rand(N, D, seed=1, dt=dt), rand(N, D, seed=2, dt=dt)
        idx = torch.rand(N, E, generator=torch.Generator().manual_seed(3)).topk(K, 1).indices.cuda()
        wt = torch.rand(N, K, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
        w_gu = rand(E, D, 2 * F, seed=5, dt=dt, scale=D ** -0.5)
        w_down = rand(E, F, D, seed=6, dt=dt, scale=F ** -0.5)
        shared = rand(N, D, seed=7, dt=dt)
        y, saved = _moe(pc, x, idx, wt, w_gu, w_down, shared, E)
        got = (y, *_moe_backward(pc, dy, x, wt, w_gu, w_down, saved))
        leaves = [t.double().requires_grad_() for t in (x, w_gu, w_down, wt)]
        X, GU, DN, WT = leaves
        out = shared.double()
        for k in range(K):
            for e in range(E):
                m = (idx[:, k] == e).nonzero().flatten()
                h = act64("swiglu", X[m] @ GU[e]) @ DN[e]
                out = out.index_add(0, m, h * WT[m, k, None])
        grads = torch.autograd.grad(out, leaves, dy.double())
        for g, want, name, tol in zip(got, (out.detach(), *grads), ("y", "dx", "dgu", "ddown", "dwt"),
                                      (fwd, bwd, bwd, bwd, bwd)):
            if name == "dwt":  # bf16 in both, as the combine takes its weights
                tol = max(tol, 2.0 ** -8)
            err = (g.double() - want).abs().max().item() / want.abs().max().item()
            assert err <= tol, f"{dtype} {name}: {err:.2e}"


def test_captured_replays_and_other_streams(pc):
    """Plan, products and gradients captured once and replayed over new inputs, with eager calls
    between the replays, equal the eager results; so does a call on another stream."""
    N, D, F, E, K = 300, 128, 64, 16, 4
    dt = torch.bfloat16
    x, dy = rand(N, D, seed=1, dt=dt), rand(N, D, seed=2, dt=dt)
    idx = torch.rand(N, E, generator=torch.Generator().manual_seed(3)).topk(K, 1).indices.cuda()
    wt = torch.rand(N, K, generator=torch.Generator().manual_seed(4)).to(dt).cuda()
    w_gu, w_down = rand(E, D, 2 * F, seed=5, dt=dt, scale=0.1), rand(E, F, D, seed=6, dt=dt, scale=0.1)

    def step():
        y, saved = _moe(pc, x, idx, wt, w_gu, w_down, None, E)
        h, pre = pc.fused_linear_forward(x, w_gu[0], None, "gelu", save_pre=True)
        lin = pc.fused_linear_backward(h, x, w_gu[0], pre, "gelu", bias=True)
        return [y, *_moe_backward(pc, dy, x, wt, w_gu, w_down, saved), h, *lin]

    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    side.synchronize()
    for a, b in zip(step(), other):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(4):
        x.copy_(rand(N, D, seed=10 + r, dt=dt))
        idx.copy_(torch.rand(N, E, generator=torch.Generator().manual_seed(20 + r)).topk(K, 1).indices)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_offsets_past_32_bits(pc):
    """Rows whose elements lie past 2^31 in x and in y."""
    dt = torch.bfloat16
    R, I, O = 2 ** 21 + 70, 1024, 1032
    x = torch.empty(R, I, dtype=dt, device="cuda")
    names = torch.tensor([R - 1, 0, R - 33, 2 ** 21, 5], dtype=torch.int32).cuda()
    x[names.long()] = rand(5, I, seed=1, dt=dt)
    w = rand(1, I, O, seed=2, dt=dt, scale=I ** -0.5)
    off = torch.tensor([0, 5], dtype=torch.int32).cuda()
    y = pc.grouped_linear_forward(x, w, off, names)
    check_forward(y, None, x[names.long()], w[0], None, "none", dt)
    dy = rand(5, O, seed=3, dt=dt)
    dx, dw, _ = pc.grouped_linear_backward(dy, x, w, off, names)
    check_backward(dx, dw[0], None, dy, x[names.long()], w[0], dy, "none", dt)
    del x, dx, y
    x = rand(64, 64, seed=4, dt=dt).repeat(2 ** 15 + 1, 1)
    w = rand(1032, 64, seed=5, dt=dt)
    y = pc.fused_linear_forward(x, w)
    assert y.numel() > 2 ** 31
    check_forward(y[-64:], None, x[-64:], w.t(), None, "none", dt)
    assert torch.equal(y[-64:], y[:64]) and torch.equal(y[2 ** 20:2 ** 20 + 64], y[:64])


@pytest.mark.parametrize("I", [64, 777, 4096])
@pytest.mark.parametrize("M", [3, 200])
def test_linear_fp32_small_values(pc, M, I):
    """Products far below one, from operands of 2^-55 each and of 2^-100 by 1, keep fp32's precision:
    the parts an operand is cut into, and their products, are not lost below bf16's range or
    fp32's normal numbers. Scaling by powers of two changes no bound but for subnormal
    products, each of the six per term within 2^-149, and for subnormal last parts, 2^-134."""
    for a, b in ((-55, -55), (-100, 0), (0, -100)):
        x = rand(M, I, seed=M + I, dt=torch.float32) * 2.0 ** a
        w = rand(264, I, seed=I, dt=torch.float32) * 2.0 ** b
        y = pc.fused_linear_forward(x, w)
        want = x.double() @ w.double().t()
        t = (I + 2) * U * (x.double().abs() @ w.double().abs().t()) + 6 * I * 2.0 ** -149
        t += 2.0 ** -134 * (x.double().abs().sum(1, keepdim=True) + w.double().abs().sum(1))
        check(y, want, U * (want.abs() + t) + t, f"2^{a} 2^{b}")


def _forward_workspace(x, w):
    from pulsar_cuda import _lib

    return _lib.load().pulsar_fused_linear_forward_workspace_bytes(
        x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), w.stride(1), *x.shape, w.shape[0], 0,
        _lib.PULSAR_BF16 if x.dtype == torch.bfloat16 else _lib.PULSAR_F32)


@pytest.mark.parametrize("dtype,M,I,O", [
    ("bf16", 250, 4096, 4088), ("bf16", 256, 4104, 4096), ("bf16", 16000, 4096, 104),
    ("fp32", 1, 4096, 1024), ("fp32", 17, 4100, 516), ("fp32", 300, 4096, 1000), ("fp32", 2331, 2056, 1024)])
@pytest.mark.parametrize("order", ["oi", "io"])
def test_linear_split_products(pc, dtype, M, I, O, order):
    """Sums over a long k shared by workgroups: forward, and dx where d_out is the long side."""
    dt = DT[dtype]
    x, dy = rand(M, I, seed=1, dt=dt), rand(M, O, seed=4, dt=dt)
    w = rand(O, I, seed=2, dt=dt, scale=I ** -0.5)
    if order == "io":
        w = w.t().contiguous().t()
    if order == "oi" and I % 8 == 0:
        split = _forward_workspace(x, w) >= 2 * M * O * 4
        assert split or M == 16000
    b = rand(O, seed=3, dt=torch.float32)
    for act in ("none", "gelu", "relu", "swiglu"):
        res = rand(M, O // 2 if act == "swiglu" else O, seed=5, dt=dt)
        y, pre = pc.fused_linear_forward(x, w, b, act, res, save_pre=True)
        check_forward(y, pre, x, w.t(), b, act, dt, res, what=act)
        again = pc.fused_linear_forward(x, w, b, act, res)
        assert torch.equal(y, again)
    y = pc.fused_linear_forward(x, w)
    check_forward(y, None, x, w.t(), None, "none", dt)
    # the same matrix the other way round: its d_out is long, and dx's sum over it is split
    ww, g = w.t(), rand(M, I, seed=6, dt=dt)
    dx, dw, db = pc.fused_linear_backward(g, dy, ww, bias=True)
    check_backward(dx, dw.t(), db, g, dy, ww.t(), g, "none", dt)


@pytest.mark.parametrize("M", [17, 300])
def test_linear_fp32_infinities_in_splits(pc, M):
    """An infinite or NaN operand in one split's part of the sum reaches its rows or columns, and only those."""
    I, O = 4096, 520
    x, w = rand(M, I, seed=1, dt=torch.float32), rand(O, I, seed=2, dt=torch.float32)
    clean = pc.fused_linear_forward(x, w)
    x[3, 4000] = math.inf
    x[5, 7] = math.nan
    w[11, 2000] = -math.inf
    y = pc.fused_linear_forward(x, w)
    want = x.double() @ w.double().t()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[odd].nan_to_num(1, 2, 3), want[odd].float().nan_to_num(1, 2, 3))
    rows = torch.ones(M, dtype=torch.bool, device="cuda")
    rows[[3, 5]] = False
    cols = torch.arange(O, device="cuda") != 11
    t = (I + 2) * U * (x[rows].double().abs() @ w[cols].double().abs().t())
    check(y[rows][:, cols], want[rows][:, cols], U * (want[rows][:, cols].abs() + t) + t, "finite")
    assert torch.isfinite(clean).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("order", ["io", "oi"])
def test_grouped_odd_widths_of_few_experts(pc, order, act, dtype):
    """Odd rows are copied into padded ones, of the groups that have rows only: most have none, and
    the weights of those are NaN."""
    dt = DT[dtype]
    E, I, O, counts = 70, 37, 42, {0: 3, 5: 1, 64: 20, 69: 2}
    off = torch.tensor([0] + [counts.get(e, 0) for e in range(E)]).cumsum(0).to(torch.int32).cuda()
    M = int(off[-1]) + 4  # and rows of no group
    w = torch.full((E, I, O), math.nan, dtype=dt, device="cuda")
    for e in counts:
        w[e] = rand(I, O, seed=e, dt=dt, scale=I ** -0.5)
    if order == "oi":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    cols = O // 2 if act == "swiglu" else O
    x, dy = rand(M, I, seed=101, dt=dt), rand(M, cols, seed=102, dt=dt)
    y, pre = pc.grouped_linear_forward(x, w, off, activation=act, save_pre=True)
    dx, dw, db = pc.grouped_linear_backward(dy, x, w, off, None, pre, act, True)
    start = 0
    for e in range(E):
        n = counts.get(e, 0)
        r = slice(start, start + n)
        if n:
            check_forward(y[r], pre[r], x[r], w[e], None, act, dt, what=f"group {e}")
            check_backward(dx[r], dw[e], db[e], dy[r], x[r], w[e], pre[r], act, dt, what=f"group {e}")
        else:
            assert not dw[e].any() and not db[e].any()
        start += n
    assert not y[start:].any() and not pre[start:].any() and not dx[start:].any()
