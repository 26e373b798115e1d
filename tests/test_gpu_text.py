"""GPU numerics of the text operators (linear, gated linear, layer norm, embedding) against plain
float64 implementations, forward and backward, through the public functions.

Tolerances are relative 2-norms. A result rounded once to a type with unit roundoff u (bf16 2^-8,
fp16 2^-11) is off by at most u in each value; a gradient product also reads dz rounded once, so
its terms are off by u each, and the two add up to at most 2 u. fp32 results of sums over at most
n values accumulate at most ~ n / 2 roundings of 2^-24 in the worst case and sqrt(n) of them in
random order; n <= 2^14 here, so 2^-24 * 2^7 * 2 bounds them with room for the few operations around
the sum."""

from __future__ import annotations

import math
import zlib

import pytest
import torch

from diffucore_b200 import _lib, kernels, text

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -16}


def close(got: torch.Tensor, want: torch.Tensor, roundings: int = 1) -> None:
    assert got.shape == want.shape
    assert got.is_contiguous()
    a, b = got.double(), want.double()
    scale = b.norm().item()
    err = (a - b).norm().item()
    assert err <= roundings * UNIT[got.dtype] * scale + 1e-30, (err / max(scale, 1e-30), got.dtype)


def act64(kind, z):
    if kind is None:
        return z
    if kind == "relu":
        return z.clamp_min(0)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def rand(gen, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(DEV)


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


@pytest.fixture(params=["auto", "0", "1"])
def kernel_choice(request, monkeypatch):
    """The rule's choice, the cluster kernel and the pair kernel: each takes every shape."""
    if request.param == "auto":
        monkeypatch.delenv("DC_HGEMM_PAIR", raising=False)
    else:
        monkeypatch.setenv("DC_HGEMM_PAIR", request.param)


@pytest.fixture(autouse=True)
def no_device_error():
    yield
    assert _lib.device_error() == 0


SHAPES = [(1, 64, 64), (1, 4096, 512), (3, 8, 8), (17, 1, 40), (127, 129, 63), (128, 128, 128), (130, 257, 72),
          (255, 96, 1000), (256, 256, 64), (300, 520, 333), (777, 640, 2048), (1232, 1280, 640)]
SMALL = [(1, 64, 64), (2, 8, 8), (17, 1, 40), (127, 129, 63), (300, 520, 333), (1025, 256, 192)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_linear_forward(kernel_choice, M, N, K, act):
    g = gen(M, N, K)
    x, w, b = rand(g, M, K), rand(g, N, K, std=K ** -0.5), rand(g, N)
    r = rand(g, M, N)
    z = x.double() @ w.double().t()
    close(text.linear(x, w, activation=act), act64(act, z))
    close(text.linear(x, w, b, activation=act, residual=r), act64(act, z + b.double()) + r.double())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_linear_activations_and_types(kernel_choice, dtype, act):
    g = gen(dtype, act)
    M, N, K = 200, 136, 96
    x, w, b, r = (rand(g, *s, dtype=dtype) for s in ((M, K), (N, K), (N,), (M, N)))
    close(text.linear(x, w, b, activation=act, residual=r),
          act64(act, x.double() @ w.double().t() + b.double()) + r.double())


@pytest.mark.parametrize("M,N,K", SMALL)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_backward(kernel_choice, M, N, K, act, dtype):
    g = gen(M, N, K, act)
    ts = [rand(g, M, K, dtype=dtype), rand(g, N, K, dtype=dtype, std=K ** -0.5), rand(g, N, dtype=dtype),
          rand(g, M, N, dtype=dtype)]
    dy = rand(g, M, N, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in ts]
    y = text.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    got = torch.autograd.grad(y, leaves, dy)
    x, w, b, r = (t.double().requires_grad_() for t in ts)
    want_y = act64(act, x @ w.t() + b) + r
    want = torch.autograd.grad(want_y, (x, w, b, r), dy.double())
    close(y.detach(), want_y.detach())
    for a, e in zip(got, want):
        close(a, e, 2)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_forward(kernel_choice, M, N, K, act):
    g = gen(M, N, K, 1)
    x, wg, wu = rand(g, M, K), rand(g, N, K, std=K ** -0.5), rand(g, N, K, std=K ** -0.5)
    bg, bu = rand(g, N), rand(g, N)
    zg, zu = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    close(text.gated_linear(x, wg, wu, activation=act), act64(act, zg) * zu)
    close(text.gated_linear(x, wg, wu, bg, bu, activation=act), act64(act, zg + bg.double()) * (zu + bu.double()))
    close(text.gated_linear(x, wg, wu, None, bu, activation=act), act64(act, zg) * (zu + bu.double()))


@pytest.mark.parametrize("M,N,K", SMALL)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh", "relu", None])
def test_gated_backward(kernel_choice, M, N, K, act):
    g = gen(M, N, K, act, 2)
    ts = [rand(g, M, K), rand(g, N, K, std=K ** -0.5), rand(g, N, K, std=K ** -0.5), rand(g, N), rand(g, N)]
    dh = rand(g, M, N)
    leaves = [t.clone().requires_grad_() for t in ts]
    h = text.gated_linear(*leaves, activation=act)
    got = torch.autograd.grad(h, leaves, dh)
    d = [t.double().requires_grad_() for t in ts]
    want_h = act64(act, d[0] @ d[1].t() + d[3]) * (d[0] @ d[2].t() + d[4])
    want = torch.autograd.grad(want_h, d, dh.double())
    close(h.detach(), want_h.detach())
    for a, e in zip(got, want):
        close(a, e, 2)


def test_gradient_against_differences():
    """The directional derivative of a fp32-read loss against central differences of the float64
    formula evaluated at the same (16-bit) point."""
    g = gen("differences")
    M, N, K = 24, 40, 32
    ts = [rand(g, M, K, dtype=torch.float16), rand(g, N, K, dtype=torch.float16, std=K ** -0.5),
          rand(g, N, K, dtype=torch.float16, std=K ** -0.5), rand(g, N, dtype=torch.float16),
          rand(g, N, dtype=torch.float16)]
    dh = rand(g, M, N, dtype=torch.float16)
    leaves = [t.clone().requires_grad_() for t in ts]
    grads = torch.autograd.grad(text.gated_linear(*leaves, activation="gelu"), leaves, dh)
    d64 = [t.double() for t in ts]

    def loss(p):
        return ((act64("gelu", p[0] @ p[1].t() + p[3]) * (p[0] @ p[2].t() + p[4])) * dh.double()).sum()

    for i, gr in enumerate(grads):
        v = torch.randn(ts[i].shape, generator=g).double().to(DEV)
        eps = 1e-5
        hi = loss([t + eps * v if j == i else t for j, t in enumerate(d64)])
        lo = loss([t - eps * v if j == i else t for j, t in enumerate(d64)])
        diff = ((hi - lo) / (2 * eps)).item()
        got = (gr.double() * v).sum().item()
        # each gradient value carries at most two roundings of the type: |error| <= 2 u ||g|| ||v||
        assert abs(got - diff) <= 2 * UNIT[torch.float16] * gr.double().norm().item() * v.norm().item()


@pytest.mark.parametrize("needs", range(1, 16))
def test_linear_partial_gradients(needs):
    g = gen("partial")
    ts = [rand(g, 40, 48), rand(g, 56, 48), rand(g, 56), rand(g, 40, 56)]
    dy = rand(g, 40, 56)
    leaves = [t.clone().requires_grad_(bool(needs >> i & 1)) for i, t in enumerate(ts)]
    full = [t.clone().requires_grad_() for t in ts]
    text.linear(leaves[0], leaves[1], leaves[2], activation="silu", residual=leaves[3]).backward(dy)
    text.linear(full[0], full[1], full[2], activation="silu", residual=full[3]).backward(dy)
    for a, b in zip(leaves, full):
        if a.requires_grad:
            assert torch.equal(a.grad, b.grad)
        else:
            assert a.grad is None


@pytest.mark.parametrize("needs", range(1, 32))
def test_gated_partial_gradients(needs):
    g = gen("partial gated")
    ts = [rand(g, 40, 48), rand(g, 56, 48), rand(g, 56, 48), rand(g, 56), rand(g, 56)]
    dh = rand(g, 40, 56)
    leaves = [t.clone().requires_grad_(bool(needs >> i & 1)) for i, t in enumerate(ts)]
    full = [t.clone().requires_grad_() for t in ts]
    text.gated_linear(*leaves).backward(dh)
    text.gated_linear(*full).backward(dh)
    for a, b in zip(leaves, full):
        if a.requires_grad:
            assert torch.equal(a.grad, b.grad)
        else:
            assert a.grad is None


def test_strides_broadcast_and_leading_dims(kernel_choice):
    g = gen("strides")
    base, wbase = rand(g, 6, 50, 200), rand(g, 200, 90)
    x = base[:, :, 3:93]                                   # odd offset, row stride 200
    w = wbase[:150, 0:90]
    wt = rand(g, 90, 150).t()                              # inner stride 150
    row = rand(g, 150)
    for weight in (w, wt):
        want = x.double() @ weight.double().t() + row.double()
        close(text.linear(x, weight, residual=row.expand(6, 50, 150)), want)
        close(text.linear(x, weight, row), want)
    xl, wl, rl = (t.detach().clone().requires_grad_() for t in (base, wt, row))
    y = text.linear(xl[:, :, 3:93], wl, residual=rl.expand(6, 50, 150), activation="silu")
    y.sum().backward()                                     # an expanded gradient
    xd, wd, rd = (t.detach().double().requires_grad_() for t in (base, wt, row))
    (act64("silu", xd[:, :, 3:93] @ wd.t()) + rd.expand(6, 50, 150)).sum().backward()
    for a, e in ((xl, xd), (wl, wd)):
        close(a.grad.contiguous(), e.grad, 2)
    close(rl.grad, rd.grad, 3)                             # summed by autograd in bf16


def test_empty_and_repeatable():
    g = gen("empty")
    w, b = rand(g, 24, 16).requires_grad_(), rand(g, 24).requires_grad_()
    x = torch.empty(0, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = text.linear(x, w, b, activation="silu")
    assert y.shape == (0, 24)
    y.sum().backward()
    assert x.grad.shape == (0, 16) and not w.grad.any() and not b.grad.any()
    h = text.gated_linear(x, w, w, b, b)
    assert h.shape == (0, 24)
    assert all(not t.any() for t in torch.autograd.grad(h.sum(), (w, b)))
    x = rand(g, 3000, 16)
    first = torch.autograd.grad(text.linear(x, w, b, activation="gelu").sum(), (w, b))
    again = torch.autograd.grad(text.linear(x, w, b, activation="gelu").sum(), (w, b))
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_infinities_and_nan_stay_in_their_rows():
    """A row of x with an infinity or NaN spoils its own row of y and no other."""
    g = gen("inf")
    x, w = rand(g, 300, 64), rand(g, 200, 64)
    clean = text.linear(x, w)
    x[7, 3], x[290, 5] = float("inf"), float("nan")
    y = text.linear(x, w)
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[7] = keep[290] = False
    assert torch.equal(y[keep], clean[keep])
    assert y[290].isnan().all() and not y[7].isfinite().any()
    big = torch.full((1, 64), -3e38, device=DEV, dtype=torch.bfloat16)
    one = torch.zeros(8, 64, device=DEV, dtype=torch.bfloat16)
    one[:, 0] = 1
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        leaf = big.clone().requires_grad_()
        y = text.linear(leaf, one, activation=act)
        assert not y.any(), act
        assert not torch.autograd.grad(y.sum(), leaf)[0].any(), act


def test_side_stream():
    g = gen("stream")
    x, w = rand(g, 500, 256), rand(g, 300, 256)
    want = text.linear(x, w, activation="gelu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = text.linear(x, w, activation="gelu")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


# ─── layer norm ─────────────────────────────────────────────────────────────────────────

def norm64(x, w, b, eps=1e-5):
    c = x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    y = y if w is None else y * w
    return y if b is None else y + b


@pytest.mark.parametrize("M,D", [(1, 1), (1, 8), (3, 33), (5, 256), (9, 257), (8, 512), (700, 768), (2, 1023), (4, 1024),
                                 (300, 1280), (31, 2047), (7, 2048), (513, 4096), (3, 4104), (2, 8192), (5, 8193),
                                 (40, 10000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("affine", ["same", "fp32", "none"])
def test_layer_norm(M, D, dtype, affine):
    g = gen(M, D, affine)
    x, dy = rand(g, M, D, dtype=dtype, std=2.0) + 1.5, rand(g, M, D, dtype=dtype)
    kind = torch.float32 if affine == "fp32" else dtype
    w, b = (None, None) if affine == "none" else (rand(g, D, dtype=kind) + 1, rand(g, D, dtype=kind))
    leaves = [t.clone().requires_grad_() for t in (x, w, b) if t is not None]
    y = text.layer_norm(*leaves)
    assert torch.equal(y, text.layer_norm(x, w, b))
    got = torch.autograd.grad(y, leaves, dy)
    d = [t.double().requires_grad_() for t in (x, w, b) if t is not None]
    want_y = norm64(d[0], *(d[1:] or (None, None)))
    want = torch.autograd.grad(want_y, d, dy.double())
    if D == 1:                                             # xhat is 0: y = b, dx = 0
        assert torch.equal(y, torch.zeros_like(y) if b is None else b.to(dtype).expand(M, 1))
        assert not got[0].any()
        return
    close(y.detach(), want_y.detach())
    for a, e in zip(got, want):
        close(a, e)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,D", [(1300, 65), (1301, 999), (2, 2047), (17, 2047), (1201, 2049), (1190, 4095), (1185, 1028),
                                 (1200, 300)])
def test_layer_norm_rows_at_any_offset(M, D, dtype):
    """Rows that start anywhere in a 16-byte window, alike in x, dy and dx (contiguous tensors, and ones
    that begin off a boundary) and not alike (a view with another row pitch)."""
    g = gen(M, D, "offset rows")
    w, b = rand(g, D, dtype=dtype) + 1, rand(g, D, dtype=dtype)

    def check(x, dy):
        leaves = [x.detach().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
        y = text.layer_norm(*leaves)
        got = torch.autograd.grad(y, leaves, dy)
        d = [t.detach().double().requires_grad_() for t in leaves]
        want_y = norm64(*d)
        close(y.detach(), want_y.detach())
        for a, e in zip(got, torch.autograd.grad(want_y, d, dy.double())):
            close(a.contiguous(), e)

    x, dy = rand(g, M, D, dtype=dtype, std=2.0) + 0.5, rand(g, M, D, dtype=dtype)
    check(x, dy)
    off = rand(g, M * D + 3, dtype=dtype)
    check(off[3:].view(M, D), dy)
    wide = rand(g, M, D + 5, dtype=dtype)
    check(wide[:, 1:D + 1], dy)
    check(x, wide[:, 2:D + 2])


def test_layer_norm_views_and_constant_rows():
    g = gen("norm views")
    base = rand(g, 6, 9, 300)
    x = base[:, 1:8, 5:261]                                # misaligned rows
    close(text.layer_norm(x, eps=1e-3), norm64(x.double(), None, None, 1e-3))
    const = torch.full((4, 128), 3.0, device=DEV, dtype=torch.bfloat16)
    assert not text.layer_norm(const).any()
    leaf = const.clone().requires_grad_()
    dx, = torch.autograd.grad(text.layer_norm(leaf), leaf, torch.ones_like(leaf))
    assert torch.isfinite(dx.float()).all()
    w32, b16 = torch.randn(128, device=DEV).requires_grad_(), rand(g, 128).requires_grad_()   # mixed types
    y = text.layer_norm(rand(g, 50, 128), w32, b16)
    dw, db = torch.autograd.grad(y, (w32, b16), torch.ones_like(y))
    assert dw.dtype == torch.float32 and db.dtype == torch.bfloat16
    assert torch.equal(db, torch.full_like(db, 50))
    assert text.layer_norm(torch.empty(0, 64, device=DEV)).shape == (0, 64)


def test_layer_norm_large_offset():
    """A mean far above the deviations: squared deviations, not a difference of squares."""
    g = gen("offset")
    x = torch.randn(64, 1024, generator=g).to(DEV) + 4096.0
    want = norm64(x.double(), None, None)
    # x itself is given to 2^-11 relative to a deviation of 1; the mean in fp32 to 4096 * 2^-24
    assert (text.layer_norm(x).double() - want).abs().max().item() < 4096 * 2 ** -22


def test_graph_capture_and_replay():
    """The calls enqueue work only: a training step captured once gives the same results when replayed
    on new inputs."""
    g = gen("graph")
    x, w, b = (rand(g, *s).requires_grad_() for s in ((300, 128), (256, 128), (256,)))
    nw = rand(g, 256).requires_grad_()
    ids = torch.randint(0, 300, (500,), device=DEV)
    dy = rand(g, 500, 256)

    def step():
        table = text.layer_norm(text.linear(x, w, b, activation="gelu"), nw)
        return torch.autograd.grad(text.embedding(ids, table), (x, w, b, nw), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(rand(g, 300, 128))
        ids.copy_(torch.randint(0, 300, (500,), device=DEV))
    graph.replay()
    got = [t.clone() for t in out]
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, out))
    assert all(torch.equal(p, q) for p, q in zip(got, step()))


# ─── embedding ──────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 10, 64), (7, 3, 40), (77, 1000, 768), (1000, 5, 72), (33, 70000, 8),
                                   (5000, 300, 129), (8192, 4000, 64), (8193, 4000, 64), (20000, 511, 33),
                                   (20000, 512, 16), (30000, 600000, 8), (100, 600000, 24), (9000, 1, 264)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("padding", [None, 0])
def test_embedding(T, V, D, dtype, padding):
    g = gen(T, V, D)
    table = rand(g, V, D, dtype=dtype).requires_grad_()
    ids = (torch.rand(T, generator=g) ** 3 * V).long().clamp_max(V - 1).to(DEV)
    dy = rand(g, T, D, dtype=dtype)
    scale = 1.7
    y = text.embedding(ids, table, scale=scale, padding_idx=padding)
    assert torch.equal(y, (table.detach()[ids].float() * scale).to(dtype))
    assert torch.equal(y, text.embedding(ids.int(), table.detach(), scale=scale))
    got, = torch.autograd.grad(y, table, dy)
    want = torch.zeros(V, D, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double() * scale)
    if padding is not None:
        want[padding] = 0
        assert not got[padding].any()
    close(got, want)
    assert not got[torch.bincount(ids, minlength=V) == 0].any()
    again, = torch.autograd.grad(text.embedding(ids, table, scale=scale, padding_idx=padding), table, dy)
    assert torch.equal(got, again)


def test_embedding_one_row_for_all_and_views():
    g = gen("same id")
    for T in (300, 8000, 30000):
        ids = torch.full((T,), 3, device=DEV)
        table = rand(g, 5, 48, dtype=torch.float32).requires_grad_()
        dy = rand(g, T, 48, dtype=torch.float32)
        got, = torch.autograd.grad(text.embedding(ids, table), table, dy)
        want = torch.zeros(5, 48, dtype=torch.float64, device=DEV)
        want[3] = dy.double().sum(0)
        close(got, want)
        one, = torch.autograd.grad(text.embedding(ids, table), table, torch.ones(1, 1, device=DEV).expand(T, 48))
        assert torch.equal(one[3], torch.full((48,), float(T), device=DEV))
    wide = rand(g, 20, 100)
    ids = torch.tensor([[1, 19], [0, 1]], device=DEV)
    assert torch.equal(text.embedding(ids, wide[:, 3:67]), wide[:, 3:67][ids])
    assert torch.equal(text.embedding(ids.t(), wide.t()[:50].t()), wide[:, :50][ids.t()])
    assert text.embedding(ids[:0], wide).shape == (0, 2, 100)
    leaf = wide.clone().requires_grad_()
    assert not torch.autograd.grad(text.embedding(ids[:0], leaf).sum(), leaf)[0].any()


def test_embedding_id_outside_the_table():
    g = gen("outside")
    table = rand(g, 10, 32).requires_grad_()
    ids = torch.tensor([3, 10, -1, 9, 1 << 40], device=DEV)
    assert _lib.device_error() == 0
    y = text.embedding(ids, table)
    assert _lib.device_error() == 3
    ok = torch.tensor([0, 3], device=DEV)
    assert torch.equal(y[ok], table[ids[ok]]) and not y[[1, 2, 4]].any()
    dy = torch.ones_like(y)
    got, = torch.autograd.grad(y, table, dy)
    want = torch.zeros_like(table)
    want[3] = want[9] = 1
    assert torch.equal(got, want)


# ─── refusals ───────────────────────────────────────────────────────────────────────────

def test_refusals():
    g = gen("refusals")
    x, w = rand(g, 4, 16), rand(g, 8, 16)
    with pytest.raises(ValueError, match="width"):
        text.linear(rand(g, 4, 15), w)
    with pytest.raises(TypeError, match="dtype"):
        text.linear(x.float(), w.float())
    with pytest.raises(TypeError, match="expected"):
        text.linear(x, w.half())
    with pytest.raises(TypeError, match="bias"):
        text.linear(x, w, torch.zeros(8, device=DEV))
    with pytest.raises(ValueError, match="bias"):
        text.linear(x, w, rand(g, 9))
    with pytest.raises(ValueError, match="residual"):
        text.linear(x, w, residual=rand(g, 1, 8))
    with pytest.raises(ValueError, match="activation"):
        text.linear(x, w, activation="swish")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        text.linear(x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="do not match"):
        text.gated_linear(x, w, rand(g, 9, 16))
    with pytest.raises(RuntimeError, match="bad shape"):
        text.linear(rand(g, 4, 16)[:, :0], w[:, :0])
    with pytest.raises(TypeError, match="weight"):
        text.layer_norm(x, rand(g, 16, dtype=torch.float16))
    with pytest.raises(ValueError, match="weight"):
        text.layer_norm(x, rand(g, 15))
    with pytest.raises(TypeError, match="ids"):
        text.embedding(torch.zeros(3, device=DEV), w)
    with pytest.raises(TypeError, match="ids"):
        text.embedding(torch.zeros(3, dtype=torch.long), w)
    with pytest.raises(ValueError, match="padding_idx"):
        text.embedding(torch.zeros(3, dtype=torch.long, device=DEV), w, padding_idx=8)
    with pytest.raises(ValueError, match="rows"):
        kernels.embedding_grad(x, torch.zeros(3, dtype=torch.long, device=DEV), 8)


def test_create_graph_gives_gradients_that_cannot_be_differentiated_again():
    g = gen("twice")
    x, w = rand(g, 6, 16).requires_grad_(), rand(g, 8, 16).requires_grad_()
    plain, = torch.autograd.grad(text.linear(x, w, activation="silu").sum(), x)
    dx, = torch.autograd.grad(text.linear(x, w, activation="silu").sum(), x, create_graph=True)
    assert torch.equal(dx.detach(), plain)
    with pytest.raises(RuntimeError):                      # no path back to x
        torch.autograd.grad(dx.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        dx.sum().backward()


def test_operand_changed_in_place_is_noticed():
    g = gen("in place")
    x, w = rand(g, 6, 16).requires_grad_(), rand(g, 8, 16).requires_grad_()
    y = text.linear(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [5, 1024])
def test_activation_and_derivative_over_the_whole_range(act, dtype, rows):
    """Value by value against float64, for z from the type's smallest to beyond where the activation is
    z or 0: weights that are the identity make z = x, and dx = dy act'(z) (here dy = 1). The result is
    the rounding of a value within the error of the fp32 arithmetic, so it lies between the roundings
    of that interval's ends. The error: the tail polynomial 0.75e-7, and the exponential and the
    reciprocal (2 units each plus 1.2 per unit of the exponent, on a probability <= 1/2) under 4e-7
    together; times |z| in the value, and once more for z phi(z) in the derivative."""
    n = rows * 64
    mags = torch.logspace(-6, math.log10(40.0), n // 2 - 1, dtype=torch.float64)
    z = torch.cat([-mags.flip(0), torch.zeros(2, dtype=torch.float64), mags]).to(dtype).view(rows, 64).to(DEV)
    eye = torch.eye(64, dtype=dtype, device=DEV)
    x = z.clone().requires_grad_()
    y = text.linear(x, eye, activation=act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    zd = z.double().requires_grad_()
    want = act64(act, zd)
    want_dx, = torch.autograd.grad(want.sum(), zd)
    size = zd.detach().abs()
    for got, exact, err in ((y.detach(), want.detach(), 5e-7 * size), (dx, want_dx, 1e-6 * (1 + size))):
        assert ((got >= (exact - err).to(dtype)) & (got <= (exact + err).to(dtype))).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 7), (3, 8), (5, 9), (40, 17), (7, 4097), (1000, 333)])
def test_operand_rows_of_any_alignment(rows, cols, dtype):
    """Exact copies, zeros behind them, whatever the offset and the pitch; nothing outside the view is
    read: the values around it are NaN."""
    g = gen(rows, cols, dtype)
    for offset in range(4):
        for pitch in (cols, cols + 1, cols + 2, cols + 5):
            store = torch.full((offset + rows * pitch + 3,), float("nan"), dtype=dtype, device=DEV)
            view = store[offset:offset + rows * pitch].as_strided((rows, cols), (pitch, 1))
            view.copy_(rand(g, rows, cols, dtype=dtype))
            m = kernels.matrix_operand(view)
            assert torch.equal(m, view) and m.data_ptr() % 16 == 0
            if m.data_ptr() != view.data_ptr():
                wide = m.as_strided((rows, m.stride(0)), (m.stride(0), 1))
                assert wide.shape[1] % 8 == 0 and (wide[:, cols:] == 0).all()
    shared = rand(g, 1, cols, dtype=dtype).expand(rows, cols)
    assert torch.equal(kernels.matrix_operand(shared), shared)


@pytest.mark.parametrize("D", [4, 8, 16, 32, 40, 64, 128, 200, 256, 264, 512, 520, 640, 768, 1152, 1536, 2560, 3008, 4160,
                               6144, 8200, 12288, 601, 1201, 2301, 5001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,affine", [(1, "same"), (1290, "same"), (1290, "fp32")])
def test_layer_norm_widths(M, D, dtype, affine):
    """Every width's launch shape, for one row and for more rows than there are row groups on the GPU: the
    last of them are partly empty."""
    M = M if M == 1 or D > 512 else 20011
    test_layer_norm(M, D, dtype, affine)


@pytest.mark.parametrize("D", [64, 96, 512])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_norm_narrow_views_and_bad_rows(D, dtype):
    """Row pitches of heads inside a wider projection; a row of NaN or infinities stays in its row of y
    and dx, whatever rows share its warp."""
    g = gen("heads", D, dtype)
    wide, dys = rand(g, 300, 3 * D, dtype=dtype), rand(g, 300, 2 * D, dtype=dtype)
    w, b = rand(g, D, dtype=dtype), rand(g, D, dtype=dtype)
    x, dy = wide[:, D:2 * D], dys[:, D:]
    leaf = x.detach().clone().requires_grad_()
    want = text.layer_norm(leaf, w, b)
    want_dx, = torch.autograd.grad(want, leaf, dy.contiguous())
    view = x.detach().requires_grad_()
    got = text.layer_norm(view, w, b)
    got_dx, = torch.autograd.grad(got, view, dy)
    assert torch.equal(got, want) and torch.equal(got_dx, want_dx)
    bad = x.clone()
    bad[7, 3], bad[100, 0], bad[299, D - 1] = float("nan"), float("inf"), -float("inf")
    leaf = bad.requires_grad_()
    y = text.layer_norm(leaf, w, b)
    dx, = torch.autograd.grad(y, leaf, dy)
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[[7, 100, 299]] = False
    assert torch.equal(y[keep], want[keep]) and torch.equal(dx[keep], want_dx[keep])
    assert y[~keep].isnan().any(-1).all() and dx[~keep].isnan().any(-1).all()
