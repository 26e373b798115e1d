"""GPU: text operators on tensors of more than 2^31 values, and on two streams at once. Whole numbers
where sums are compared, so that they are exact whatever their order."""

from __future__ import annotations

import pytest
import torch

from diffucore_b200 import device_error, text

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def clean():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GiB of free device memory")
    yield
    torch.cuda.empty_cache()
    assert device_error() == 0


def whole(*shape, most=2):
    t = torch.empty(*shape, device=DEV, dtype=BF16)
    for part in t.split(1 << 17):                            # randint's int64 stays small
        part.copy_(torch.randint(-most, most + 1, part.shape, device=DEV))
    return t


def some_rows(rows, width):
    """The first and the last rows, and those where offsets pass 2^31 and 2^32 bytes and 2^31 values."""
    picks = [torch.arange(40), torch.arange(rows - 40, rows)]
    for at in ((1 << 30) // width, (1 << 31) // width):
        picks.append(torch.arange(at - 3, min(rows, at + 4)))
    return torch.cat(picks).clamp(0, rows - 1).to(DEV)


def sums(a, b):
    """a.T @ b in float64, in parts."""
    total = 0
    for p, q in zip(a.split(1 << 16), b.split(1 << 16)):
        total = total + p.double().t() @ q.double()
    return total


@pytest.mark.parametrize("N,K", [(4096, 64), (64, 4096), (4099, 40)])
def test_linear(N, K):
    M = (1 << 31) // max(N, K) + 3000
    x, w, b = (t.requires_grad_() for t in (whole(M, K, most=1), whole(N, K, most=1), whole(N)))
    y = text.linear(x, w, b, activation="relu")
    dy = whole(M, N, most=1)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        r = some_rows(M, max(N, K))
        z = x[r].double() @ w.double().t() + b.double()
        assert torch.equal(y[r], z.clamp_min(0).to(BF16))
        assert torch.equal(dx[r], (dy[r].double() * (z > 0) @ w.double()).to(BF16))
        want_w, want_b = 0, 0
        for xs, ds in zip(x.split(1 << 16), dy.split(1 << 16)):
            dz = ds.double() * (xs.double() @ w.double().t() + b.double() > 0)
            want_w, want_b = want_w + dz.t() @ xs.double(), want_b + dz.sum(0)
        assert max(want_w.abs().max().item(), want_b.abs().max().item()) < 2 ** 24
        assert torch.equal(dw, want_w.to(BF16)) and torch.equal(db, want_b.to(BF16))


def test_gated_linear():
    M, N, K = (1 << 31) // 4096 + 3000, 4096, 64
    leaves = [t.requires_grad_() for t in (whole(M, K, most=1), whole(N, K, most=1), whole(N, K, most=1))]
    h = text.gated_linear(*leaves, activation="relu")
    dh = whole(M, N, most=1)
    dx, dwg, dwu = torch.autograd.grad(h, leaves, dh)
    with torch.no_grad():
        x, wg, wu = leaves
        r = some_rows(M, N)
        g, u, d = x[r].double() @ wg.double().t(), x[r].double() @ wu.double().t(), dh[r].double()
        assert torch.equal(h[r], (g.clamp_min(0) * u).to(BF16))
        want = d * u * (g > 0) @ wg.double() + d * g.clamp_min(0) @ wu.double()    # |dz| <= 64: exact in 16 bits
        assert torch.equal(dx[r], want.to(BF16))
        want_u = 0
        for xs, ds in zip(x.split(1 << 16), dh.split(1 << 16)):
            want_u = want_u + (ds.double() * (xs.double() @ wg.double().t()).clamp_min(0)).t() @ xs.double()
        assert want_u.abs().max().item() < 2 ** 24 and torch.equal(dwu, want_u.to(BF16))


@pytest.mark.parametrize("D", [4096, 2049, 128])
def test_layer_norm(D):
    """Against the same rows alone, which other tests compare with float64; db is a sum of whole numbers."""
    M = (1 << 31) // D + 3000
    x, dy = whole(M, D, most=100).requires_grad_(), whole(M, D, most=1)
    w, b = torch.rand(D, device=DEV).to(BF16).requires_grad_(), torch.rand(D, device=DEV).to(BF16).requires_grad_()
    y = text.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        r = some_rows(M, D)
        xs = x[r].double()
        var, mean = torch.var_mean(xs, dim=1, correction=0, keepdim=True)
        xhat = (xs - mean) * torch.rsqrt(var + 1e-5)
        a = dy[r].double() * w.double()
        want = torch.rsqrt(var + 1e-5) * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
        # one rounding to bf16 and some of fp32
        assert ((y[r].double() - (xhat * w.double() + b.double())).abs() <= 2.0 ** -8 * y[r].double().abs() + 1e-5).all()
        assert ((dx[r].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-7).all()
        total = sum(part.sum(0, dtype=torch.float64) for part in dy.split(1 << 17))
        assert total.abs().max().item() < 2 ** 24 and torch.equal(db, total.to(BF16))
        got_w = 0
        for p, q in zip(x.split(1 << 15), dy.split(1 << 15)):
            p = p.double()
            var, mean = torch.var_mean(p, dim=1, correction=0, keepdim=True)
            got_w = got_w + (q.double() * (p - mean) * torch.rsqrt(var + 1e-5)).sum(0)
        # fp32 sums: at most 2^15 terms one after another per thread, far fewer than M; random signs
        assert ((dw.double() - got_w).abs() <= 2.0 ** -8 * got_w.abs() + 2.0 ** -24 * 2 ** 8 * M ** 0.5).all()


@pytest.mark.parametrize("D", [4096, 4099])
def test_embedding(D):
    """More than 2^31 values of output and of table."""
    T = V = (1 << 31) // D + 3000
    table = whole(V, D).requires_grad_()
    ids = torch.randperm(V, device=DEV)
    ids[:1000] = V - 1
    y = text.embedding(ids, table)
    dy = whole(T, D, most=1)
    got, = torch.autograd.grad(y, table, dy)
    with torch.no_grad():
        for at in range(0, T, 1 << 16):
            assert torch.equal(y[at:at + (1 << 16)], table[ids[at:at + (1 << 16)]])
        once = torch.bincount(ids, minlength=V) == 1
        place = torch.zeros(V, dtype=torch.long, device=DEV)
        place[ids] = torch.arange(T, device=DEV)
        for at in range(0, V, 1 << 16):
            part, single = got[at:at + (1 << 16)], once[at:at + (1 << 16)]
            want = dy[place[at:at + (1 << 16)]] * single[:, None]
            if at + (1 << 16) >= V:
                part, want = part[:-1], want[:-1]
            assert torch.equal(part, want)
        assert torch.equal(got[V - 1], dy[ids == V - 1].double().sum(0).to(BF16))


def test_two_streams_at_once():
    """Products of both tiled kernels, norms and sorts that run side by side."""
    torch.manual_seed(0)
    data = []
    for n in (700, 2600):
        x, w = whole(n, 512).requires_grad_(), whole(1024, 512).requires_grad_()
        data.append((x, w, torch.randint(0, n, (9000,), device=DEV), whole(9000, 1024)))

    def step(x, w, ids, dy):
        h = text.layer_norm(text.linear(x, w, activation="silu"))
        return torch.autograd.grad(text.embedding(ids, h), (x, w), dy)

    wants = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(20):
        got = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(step(*d))
        torch.cuda.synchronize()
        for a, b in zip(got, wants):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
