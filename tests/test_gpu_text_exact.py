"""GPU: the text operators value by value.

Projections on small whole numbers: every product and every fp32 sum is exact whatever its order, so an
output is the one rounding of a whole number and has to be equal bit for bit; a single value that is
missing, stale or in a wrong place fails. Layer norm against float64 within the error of its own fp32
arithmetic, derived beside the test. Nothing outside a view is read (the values around it are NaN)
and nothing outside an output is written (guard values around it)."""

from __future__ import annotations

import pytest
import torch

from diffucore_b200 import _lib, device_error, kernels, text

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: _lib.DTYPE_F32, F16: _lib.DTYPE_F16, BF16: _lib.DTYPE_BF16}


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert device_error() == 0


def whole(*shape, dtype=BF16, most=2):
    return torch.randint(-most, most + 1, shape, device=DEV).to(dtype)


def equal(got, want64, dtype):
    """``want64`` holds whole numbers that fp32 holds exactly."""
    assert want64.abs().max().item() < 2 ** 24
    assert torch.equal(got, want64.to(dtype))


# Rows, columns and depth of a product whose 256-row tiles are more than the CTA pairs (74), so that each
# pair takes a second tile, or a third: its second accumulator, the stage phases across tiles, a second
# group of tile rows. The estimate in text_api.cu gives these tile widths to the pair kernel:
WIDTHS = [(3198, 2121, 66),                                # 128 columns
          (3343, 1303, 65), (2561, 2049, 520),             # 160
          (1832, 2932, 66), (3000, 2100, 264),             # 192
          (1613, 4048, 65),                                # 224
          (1826, 4434, 66)]                                # 256
# ... and these to the cluster kernel with the depth divided by 8, 4, 2 and 1.
SPLITS = [(64, 1024, 1024), (200, 1000, 1030), (1024, 1024, 1024), (2433, 1100, 136)]


@pytest.fixture(params=["auto", "0", "1"])
def kernel_choice(request, monkeypatch):
    if request.param == "auto":
        monkeypatch.delenv("DC_HGEMM_PAIR", raising=False)
    else:
        monkeypatch.setenv("DC_HGEMM_PAIR", request.param)


def sizes(m, n, k):
    """The size itself and one whose rows are all aligned."""
    yield m, n, k
    yield m, n // 8 * 8, (k + 7) // 8 * 8


@pytest.mark.parametrize("m,n,k", WIDTHS + SPLITS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear(kernel_choice, m, n, k, dtype):
    for M, N, K in sizes(m, n, k):
        x, w, b, r = whole(M, K, dtype=dtype), whole(N, K, dtype=dtype), whole(N, dtype=dtype), whole(M, N, dtype=dtype, most=9)
        z = x.double() @ w.double().t()
        equal(text.linear(x, w), z, dtype)
        z += b.double()
        y, kept = kernels.linear(x, w, b, "relu", r, keep_z=True)
        equal(y, z.clamp_min(0) + r.double(), dtype)
        assert torch.equal(kept[:, :N], z.float())


@pytest.mark.parametrize("m,n,k", WIDTHS + SPLITS)
def test_gated_linear(kernel_choice, m, n, k):
    for M, N, K in sizes(m, n // 2, k):
        x, wg, wu, bg, bu = whole(M, K), whole(N, K), whole(N, K), whole(N), whole(N)
        g, u = x.double() @ wg.double().t() + bg.double(), x.double() @ wu.double().t() + bu.double()
        equal(text.gated_linear(x, wg, wu, bg, bu, activation=None), g * u, BF16)
        h, zg, zu = kernels.gated_linear(x, wg, wu, bg, bu, "relu", keep_z=True)
        equal(h, g.clamp_min(0) * u, BF16)
        assert torch.equal(zg[:, :N], g.float()) and torch.equal(zu[:, :N], u.float())


@pytest.mark.parametrize("m,n,k", WIDTHS + SPLITS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_backward_products(kernel_choice, m, n, k, dtype):
    """dx [m, n] over k columns of dz, and dw [m, n] over k rows, alone and in their two-product forms."""
    for M, N, K in sizes(m, n, k):
        dz, dz1, w, w1 = (whole(*s, dtype=dtype) for s in ((M, K), (M, K), (K, N), (K, N)))
        want = dz.double() @ w.double()
        equal(kernels.linear_dx(dz, w), want, dtype)
        equal(kernels.linear_dx(dz, w, dz1, w1), want + dz1.double() @ w1.double(), dtype)
        dz, dz1, x = (whole(*s, dtype=dtype) for s in ((K, M), (K, M), (K, N)))
        wants = [d.double().t() @ x.double() for d in (dz, dz1)]
        equal(kernels.linear_dw(dz, x)[0], wants[0], dtype)
        for got, want in zip(kernels.linear_dw(dz, x, dz1), wants):
            equal(got, want, dtype)


@pytest.mark.parametrize("m,n,k", [(3198, 2121, 66), (1613, 504, 65), (7, 300, 40), (12, 301, 41)])
def test_training_step(kernel_choice, m, n, k):
    """The gated block and the dense product through autograd, dz rounded to 16 bits where it is stored."""
    x, wg, wu, bg, bu = whole(m, k), whole(n, k), whole(n, k), whole(n), whole(n)
    dy = whole(m, n, most=1)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(text.gated_linear(*leaves, activation="relu"), leaves, dy)
    xd, gd, ud, d = x.double(), wg.double(), wu.double(), dy.double()
    g, u = xd @ gd.t() + bg.double(), xd @ ud.t() + bu.double()
    dg, du = d * u * (g > 0), d * g.clamp_min(0)
    dg16, du16 = dg.to(BF16).double(), du.to(BF16).double()
    for got, want in zip(grads, (dg16 @ gd + du16 @ ud, dg16.t() @ xd, du16.t() @ xd, dg.sum(0), du.sum(0))):
        equal(got, want, BF16)
    leaves = [t.clone().requires_grad_() for t in (x, wg, bg)]
    grads = torch.autograd.grad(text.linear(*leaves, activation="relu", residual=dy), leaves, dy)
    dz = d * (g > 0)
    for got, want in zip(grads, (dz @ gd, dz.t() @ xd, dz.sum(0))):
        equal(got, want, BF16)


@pytest.mark.parametrize("M,N,K", [(1, 700, 333), (3, 64, 64), (8, 1000, 4100), (8, 17, 40), (9, 300, 200), (16, 4096, 512)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_rows(M, N, K, dtype):
    for x, w, wu in ((whole(M, K, dtype=dtype), whole(N, K, dtype=dtype), whole(N, K, dtype=dtype)),
                     (inside_nan(M, K, 1, K + 3, dtype), inside_nan(N, K, 3, K + 1, dtype), inside_nan(N, K, 0, K + 2, dtype))):
        b, r = whole(N, dtype=dtype), whole(M, N, dtype=dtype)
        g, u = x.double() @ w.double().t(), x.double() @ wu.double().t()
        equal(text.linear(x, w, b, residual=r, activation="relu"), (g + b.double()).clamp_min(0) + r.double(), dtype)
        if dtype == BF16:
            equal(text.gated_linear(x, w, wu, None, b, activation="relu"), g.clamp_min(0) * (u + b.double()), dtype)


def inside_nan(rows, cols, offset, pitch, dtype=BF16, most=2):
    """A view of whole numbers with NaN before, between and behind its rows."""
    store = torch.full((offset + rows * pitch + 9,), float("nan"), dtype=dtype, device=DEV)
    view = store[offset:offset + rows * pitch].as_strided((rows, cols), (pitch, 1))
    view.copy_(whole(rows, cols, dtype=dtype, most=most))
    return view


@pytest.mark.parametrize("N", [1, 3, 7, 8, 9, 15, 17, 511, 513, 520, 1025])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_pointwise_gradient_at_any_alignment(N, dtype):
    """All three forms; dy starts anywhere, and its rows lie close (pitch N) or apart."""
    for M in (1, 2, 3, 5, 20, 70, 1200 if N < 100 else 130):
        x, wg, wu = whole(M, 16, dtype=dtype), whole(N, 16, dtype=dtype), whole(N, 16, dtype=dtype)
        _, g, u = kernels.gated_linear(x, wg, wu, act=None, keep_z=True)
        g64, u64 = g[:, :N].double(), u[:, :N].double()
        for offset in range(4):
            for pitch in (N, N + 1, N + 2, (N + 7) // 8 * 8):
                dy = inside_nan(M, N, offset, pitch, dtype, most=3)
                d = dy.double()
                dz, dz1, db, db1 = kernels.act_grad(dy, g, u, "relu", True, True)
                wants = (d * u64 * (g64 > 0), d * g64.clamp_min(0))
                equal(dz, wants[0], dtype)
                equal(dz1, wants[1], dtype)
                equal(db, wants[0].sum(0), dtype)
                equal(db1, wants[1].sum(0), dtype)
                dz, _, db, _ = kernels.act_grad(dy, g, None, "relu", True)
                equal(dz, d * (g64 > 0), dtype)
                equal(db, (d * (g64 > 0)).sum(0), dtype)
                equal(kernels.act_grad(dy, None, None, None, True)[2], d.sum(0), dtype)


@pytest.mark.parametrize("T,V,D", [(9000, 7, 264), (20000, 511, 33), (40000, 100, 64), (60000, 50, 7), (5, 9, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_embedding_writes_its_rows_and_no_others(T, V, D, dtype):
    """Also where the last tokens are fewer than the four that a row of threads takes at once."""
    for extra in range(4):
        n = T + extra
        table = torch.randn(V, D, device=DEV).to(dtype)
        ids = torch.randint(0, V, (n,), device=DEV)
        store = torch.full((n + 8, D), 77.0, dtype=dtype, device=DEV)
        out = store[4:4 + n]
        _lib.check(_lib.load().dc_embedding(ids.data_ptr(), 1, n, table.data_ptr(), D, V, D, 2.0, out.data_ptr(), D, CODE[dtype],
                                            torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, (table.float() * 2)[ids].to(dtype))
        assert (store[:4] == 77).all() and (store[4 + n:] == 77).all()


def norm_bounds(x, w, b, dy):
    """Layer norm, dx, dw and db in float64 with the error of the kernels' fp32 arithmetic (before the
    rounding to the output's type). e = 2^-24 is one fp32 rounding; no sum over a row of up to 16384
    values adds more than 64 terms one after another (the values of a thread, then a tree).
      mean    64 e mean|x| + e |mean|
      rstd    var's sums 66 e and the mean's error squared over var, both halved by the root; rsqrt 4 e
      xhat    the mean's error times rstd, rstd's relative error and 3 roundings
      y       xhat's error times |w|, 3 roundings of its terms
      dx      rstd (a - ma - xhat mh): sums of a and a xhat as above, xhat's error, 6 roundings of its terms
      dw, db  M terms one after another at the worst"""
    e = 2.0 ** -24
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True) + 1e-5
    r = var.rsqrt()
    xhat = c * r
    d_mean = 64 * e * x.abs().mean(1, keepdim=True) + e * mean.abs()
    rho = 33 * e + 0.5 * d_mean ** 2 / var + 4 * e
    d_xhat = d_mean * r + xhat.abs() * (rho + 3 * e)
    y = xhat * w + b
    d_y = d_xhat * w.abs() + 3 * e * ((xhat * w).abs() + b.abs())
    a = dy * w
    ma, mh = a.mean(1, keepdim=True), (a * xhat).mean(1, keepdim=True)
    d_ma = 66 * e * a.abs().mean(1, keepdim=True)
    d_mh = 67 * e * (a * xhat).abs().mean(1, keepdim=True) + (a.abs() * d_xhat).mean(1, keepdim=True)
    dx = r * (a - ma - xhat * mh)
    d_dx = r * (d_ma + xhat.abs() * d_mh + d_xhat * mh.abs() + 6 * e * (a.abs() + ma.abs() + (xhat * mh).abs())) + dx.abs() * rho
    terms = x.shape[0] + 2
    dw = (dy * xhat).sum(0)
    d_dw = terms * e * (dy * xhat).abs().sum(0) + (dy.abs() * d_xhat).sum(0)
    db = dy.sum(0)
    return (y, d_y), (dx, d_dx), (dw, d_dw), (db, terms * e * dy.abs().sum(0))


@pytest.mark.parametrize("M,D", [(1, 4096), (700, 64), (1300, 65), (301, 257), (1300, 768), (1290, 1280), (33, 2047), (1201, 2049),
                                 (1185, 4096), (600, 5120), (1190, 8200), (7, 10001), (300, 16384)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layer_norm(M, D, dtype):
    x = (torch.randn(M, D, device=DEV) * 2 + 0.5).to(dtype)
    dy = torch.randn(M, D, device=DEV).to(dtype)
    w, b = (torch.randn(D, device=DEV) + 1).to(dtype), torch.randn(D, device=DEV).to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = text.layer_norm(*leaves)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    bounds = norm_bounds(x.detach().double(), w.detach().double(), b.detach().double(), dy.double())
    for value, (want, err) in zip(got, bounds):
        # between the roundings of the interval's ends; two values of fp32 may round to neighbours
        assert ((value >= (want - err).to(dtype)) & (value <= (want + err).to(dtype))).all()
