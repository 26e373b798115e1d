"""Measured cases of the text-side operators: dense and gated projections, layer norm and token
embedding, forward alone and as a training step (forward, then the gradients of every input).

``run`` computes a case in plain torch operations in fp32 (``own`` false) or through
``diffucore_b200.text`` (``own`` true); ``exact`` gives the same outputs in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one conditioning vector or one decoded token through a square projection
        dict(name="linear_token", op="linear", rows=1, k=4096, n=4096, act="none", bias=True, residual=True,
             dtype="bf16", train=False),
        # a batch of sixteen 77-token prompts through the up-projection of a 1280-wide encoder's MLP
        dict(name="linear_prompts", op="linear", rows=1232, k=1280, n=5120, act="gelu", bias=True, residual=False,
             dtype="fp16", train=False),
        # a training step of a square projection with activation and residual
        dict(name="linear_train", op="linear", rows=8192, k=4096, n=4096, act="gelu_tanh", bias=True, residual=True,
             dtype="bf16", train=True),
        # four candidate tokens through a wide gated block
        dict(name="gated_tokens", op="gated", rows=4, k=4096, n=10240, act="silu", bias=False, dtype="bf16",
             train=False),
        # one 512-token prompt of 4096-wide states
        dict(name="gated_prompt", op="gated", rows=512, k=4096, n=10240, act="gelu_tanh", bias=False, dtype="bf16",
             train=False),
        # a training step over packed prompts, an inner width that no tile divides
        dict(name="gated_train", op="gated", rows=4173, k=2048, n=5461, act="silu", bias=True, dtype="bf16",
             train=True),
        # one token's norm
        dict(name="norm_token", op="norm", rows=1, k=4096, dtype="bf16", train=False),
        # a training step over rows that no vector width divides
        dict(name="norm_ragged", op="norm", rows=10007, k=2047, dtype="fp16", train=True),
        # a training step over long packed sequences
        dict(name="norm_train", op="norm", rows=32768, k=4096, dtype="bf16", train=True),
        # one 512-token prompt looked up and scaled by sqrt(width)
        dict(name="embed_prompt", op="embed", rows=512, vocab=32128, k=4096, scale=64.0, pad=False, dtype="bf16",
             train=False),
        # learning a concept's token: a small batch of prompts, dense gradient of the table
        dict(name="embed_concept", op="embed", rows=1232, vocab=49408, k=768, scale=1.0, pad=False, dtype="bf16",
             train=True),
        # training on padded sequences: a quarter of the ids is the padding token
        dict(name="embed_train", op="embed", rows=65536, vocab=32128, k=2048, scale=1.0, pad=True, dtype="bf16",
             train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 64, sometimes of 8, sometimes odd."""
    n = _log_int(rng, lo, hi)
    kind = rng.random()
    if kind < 0.6:
        return max(64, n // 64 * 64)
    if kind < 0.8:
        return max(8, n // 8 * 8)
    return n | 1


def draw(rng):
    op = rng.choice(("linear", "gated", "norm", "embed"))
    train = rng.random() < 0.5
    if op in ("linear", "gated"):
        k, n = _width(rng, 64, 4096), _width(rng, 64, 4096 if op == "linear" else 10240)
        cap = 8192 * 4096 * 4096 if op == "linear" else 4173 * 2048 * 5461
        rows = min(_log_int(rng, 1, 8192), max(1, cap // (k * n)))
        case = dict(op=op, rows=rows, k=k, n=n, act=rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                    bias=rng.random() < 0.6, dtype=rng.choice(("bf16", "bf16", "fp16")), train=train)
        if op == "linear":
            case["residual"] = rng.random() < 0.5
        return case
    if op == "norm":
        k = _width(rng, 64, 16384)
        rows = min(_log_int(rng, 1, 65536), max(1, 32768 * 4096 // k))
        return dict(op=op, rows=rows, k=k, dtype=rng.choice(("bf16", "fp16", "fp32")), train=train)
    k, vocab = _width(rng, 64, 4096), _log_int(rng, 256, 131072)
    vocab = min(vocab, 32128 * 2048 // k)
    rows = min(_log_int(rng, 1, 65536), max(1, 65536 * 2048 // k))
    return dict(op=op, rows=rows, vocab=vocab, k=k, scale=rng.choice((1.0, round(math.sqrt(k), 3))),
                pad=rng.random() < 0.5, dtype=rng.choice(("bf16", "fp16", "fp32")), train=train)


def prepare(case, seed):
    dt, m, k, train = _DTYPES[case["dtype"]], case["rows"], case["k"], case["train"]
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)

    def normal(*shape, std=1.0, mean=0.0):
        t = torch.empty(*shape, device="cuda", dtype=torch.float32).normal_(mean, std, generator=gen)
        return t.to(dt)

    def leaf(t):
        return t.requires_grad_() if train else t

    st = dict(case=dict(case))
    if case["op"] in ("linear", "gated"):
        n = case["n"]
        st["x"] = leaf(normal(m, k))
        names = ("w",) if case["op"] == "linear" else ("w_gate", "w_up")
        for name in names:
            st[name] = leaf(normal(n, k, std=1.5 / math.sqrt(k)))
        for name in names:
            st[name.replace("w", "b", 1)] = leaf(normal(n, std=0.1)) if case["bias"] else None
        if case["op"] == "linear":
            st["residual"] = leaf(normal(m, n)) if case["residual"] else None
        if train:
            st["dy"] = normal(m, n)
    elif case["op"] == "norm":
        # hidden states: per-channel offsets and a few channels much larger than the rest
        amp = torch.ones(k, device="cuda")
        amp[torch.randint(0, k, (max(1, k // 256),), device="cuda", generator=gen)] = 12.0
        off = torch.empty(k, device="cuda").normal_(0.0, 0.5, generator=gen)
        x = torch.empty(m, k, device="cuda").normal_(0.0, 1.0, generator=gen)
        st["x"] = leaf(x.mul_(amp).add_(off).to(dt))
        st["w"] = leaf(normal(k, std=0.2, mean=1.0))
        st["b"] = leaf(normal(k, std=0.2))
        if train:
            st["dy"] = normal(m, k)
    else:
        vocab = case["vocab"]
        # token frequencies fall off steeply: a few ids make up most of a batch
        u = torch.rand(m, device="cuda", generator=gen)
        ids = (u.pow(4) * vocab).long().clamp_(max=vocab - 1)
        if case["pad"]:
            ids = torch.where(torch.rand(m, device="cuda", generator=gen) < 0.25, torch.zeros_like(ids), ids)
        st["ids"] = ids
        st["table"] = leaf(normal(vocab, k, std=0.05))
        if train:
            st["dy"] = normal(m, k)
    return st


# ------------------------------------------------------------------ the framework's operators

def _run_own(st):
    from diffucore_b200 import text
    case = st["case"]
    op = case["op"]
    if op == "linear":
        act = None if case["act"] == "none" else case["act"]
        out = text.linear(st["x"], st["w"], st["b"], activation=act, residual=st["residual"])
        names = ("x", "w", "b", "residual")
    elif op == "gated":
        act = None if case["act"] == "none" else case["act"]
        out = text.gated_linear(st["x"], st["w_gate"], st["w_up"], st["b_gate"], st["b_up"], activation=act)
        names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    elif op == "norm":
        out = text.layer_norm(st["x"], st["w"], st["b"], eps=1e-5)
        names = ("x", "w", "b")
    else:
        out = text.embedding(st["ids"], st["table"], scale=case["scale"], padding_idx=0 if case["pad"] else None)
        names = ("table",)
    res = {"y": out.detach()}
    if case["train"]:
        names = [n for n in names if st[n] is not None]
        for n, g in zip(names, torch.autograd.grad(out, [st[n] for n in names], st["dy"])):
            res["d_" + n] = g
    return res


# ------------------------------------------------------------------ plain fp32 operations

def _act(kind, z):
    """(activation, its derivative) of z."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if kind == "gelu":
        c = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
    inner = math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * z * z)
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * inner


@torch.no_grad()
def _run_plain(st):
    case = st["case"]
    op, dt, train = case["op"], _DTYPES[case["dtype"]], case["train"]
    res = {}
    if op == "linear":
        x, w = st["x"].float(), st["w"].float()
        z = x @ w.t()
        if st["b"] is not None:
            z = z + st["b"].float()
        a, da = _act(case["act"], z)
        res["y"] = (a if st["residual"] is None else a + st["residual"].float()).to(dt)
        if train:
            dz = st["dy"].float() * da
            res["d_x"], res["d_w"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
            if st["b"] is not None:
                res["d_b"] = dz.sum(0).to(dt)
            if st["residual"] is not None:
                res["d_residual"] = st["dy"]
    elif op == "gated":
        x, wg, wu = st["x"].float(), st["w_gate"].float(), st["w_up"].float()
        g, u = x @ wg.t(), x @ wu.t()
        if st["b_gate"] is not None:
            g, u = g + st["b_gate"].float(), u + st["b_up"].float()
        a, da = _act(case["act"], g)
        res["y"] = (a * u).to(dt)
        if train:
            dy = st["dy"].float()
            dg, du = dy * u * da, dy * a
            res["d_x"] = (dg @ wg + du @ wu).to(dt)
            res["d_w_gate"], res["d_w_up"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
            if st["b_gate"] is not None:
                res["d_b_gate"], res["d_b_up"] = dg.sum(0).to(dt), du.sum(0).to(dt)
    elif op == "norm":
        x, w = st["x"].float(), st["w"].float()
        c = x - x.mean(1, keepdim=True)
        rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
        xhat = c * rstd
        res["y"] = (xhat * w + st["b"].float()).to(dt)
        if train:
            dy = st["dy"].float()
            dw = dy * w
            res["d_x"] = (rstd * (dw - dw.mean(1, keepdim=True) - xhat * (dw * xhat).mean(1, keepdim=True))).to(dt)
            res["d_w"], res["d_b"] = (dy * xhat).sum(0).to(dt), dy.sum(0).to(dt)
    else:
        table, ids = st["table"], st["ids"]
        res["y"] = (table[ids].float() * case["scale"]).to(dt)
        if train:
            acc = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
            acc.index_add_(0, ids, st["dy"].float() * case["scale"])
            if case["pad"]:
                acc[0] = 0.0
            res["d_table"] = acc.to(dt)
    return res


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ 64 bits

def _act64(kind, z):
    if kind == "none":
        return z
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return z * torch.special.ndtr(z)
    return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))


def exact(case, seed):
    """The definition evaluated in float64, its gradients by differentiating that evaluation."""
    st = prepare(case, seed)
    op = case["op"]
    d = {n: t.detach().double().requires_grad_(case["train"]) for n, t in st.items()
         if isinstance(t, torch.Tensor) and n not in ("ids", "dy")}
    if op == "linear":
        names = ("x", "w", "b", "residual")
        z = torch.einsum("mk,nk->mn", d["x"], d["w"])
        y = _act64(case["act"], z + d["b"] if "b" in d else z)
        if "residual" in d:
            y = y + d["residual"]
    elif op == "gated":
        names = ("x", "w_gate", "w_up", "b_gate", "b_up")
        g = torch.einsum("mk,nk->mn", d["x"], d["w_gate"])
        u = torch.einsum("mk,nk->mn", d["x"], d["w_up"])
        if "b_gate" in d:
            g, u = g + d["b_gate"], u + d["b_up"]
        y = _act64(case["act"], g) * u
    elif op == "norm":
        names = ("x", "w", "b")
        var, mean = torch.var_mean(d["x"], dim=1, correction=0, keepdim=True)
        y = (d["x"] - mean) * torch.rsqrt(var + 1e-5) * d["w"] + d["b"]
    else:
        names = ("table",)
        y = d["table"].index_select(0, st["ids"]) * case["scale"]
    res = {"y": y.detach()}
    if case["train"]:
        names = [n for n in names if n in d]
        for n, g in zip(names, torch.autograd.grad(y, [d[n] for n in names], st["dy"].double())):
            if n == "table" and case["pad"]:
                g[0] = 0.0
            res["d_" + n] = g
    return res


def work(case):
    """Bytes with each input read and each output written once, and the products' operations."""
    m, k, e, train = case["rows"], case["k"], _BYTES[case["dtype"]], case["train"]
    op = case["op"]
    if op in ("linear", "gated"):
        n, mats = case["n"], 1 if op == "linear" else 2
        weights = mats * n * (k + (1 if case["bias"] else 0))
        has_res = bool(case.get("residual"))
        values = m * k + weights + m * n * (2 if has_res else 1)
        flops = 2.0 * mats * m * n * k
        if train:   # reads dy; writes dx and the weights' and biases' gradients
            values += m * n + m * k + weights
            flops *= 3
        return {"bytes": e * values, "flops": flops}
    if op == "norm":
        values = 2 * m * k + 2 * k
        flops = 8.0 * m * k
        if train:
            values += 2 * m * k + 2 * k
            flops += 14.0 * m * k
        return {"bytes": e * values, "flops": flops}
    # the rows of the table that are looked up: at most one per token
    values = min(m, case["vocab"]) * k + m * k
    flops = 1.0 * m * k
    if train:
        values += m * k + case["vocab"] * k
        flops += 1.0 * m * k
    return {"bytes": e * values + 8 * m, "flops": flops}
