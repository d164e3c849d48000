"""What the operators around a routed expert layer are measured on.

A layer of experts stands in a block: its input is normalised, its router is kept balanced, beside it a projection that all tokens share serves
many requests' adapters, and its result passes a dropout on its way to the sum that the next block reads.

  norm         s = residual + dropout(x), y = (s - mean) rstd weight + bias, with the rows' mean and rstd
  norm_grad    its gradients: of s (with what reaches s directly added), of x behind the dropout, of weight and bias
  dropout      residual + x keep / (1 - p), keep from a counter-based generator, never stored
  balance      experts / (choices tokens) sum_e counts[e] sum_t p[t, e], the counts and the mean probabilities (``grad``: with the gradient of the
               logits that this and the router's weights give)
  adapted      y[t] = W x[t] + scale[a] B[a] A[a] x[t] with a = ids[t], -1: none

``prepare`` makes what a program holds before the call, ``run`` makes the call: the framework's where ``own`` is true, otherwise the same
formulas in elementary operations of 32 bits.  ``exact`` is the definition in 64 bits.

The generator is Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011): the key is the seed, the
counter (column / 4, row, offset low, offset high), word j the random number of column 4 (column / 4) + j, which is kept where it is at least
p 2^32.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def listed():
    return [
        # a decoding step's rows: the residual sum and its norm in one call
        {"name": "norm_16_bf16", "kind": "norm", "rows": 16, "width": 2048, "dtype": "bf16", "param": "bf16", "residual": True, "p": 0.0, "bound": True},
        # a training batch: dropout, residual sum and norm
        {"name": "norm_16k_bf16", "kind": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "param": "f32", "residual": True, "p": 0.1, "bound": False},
        # the gradients of rows of an odd width in 32 bits
        {"name": "norm_grad_4k_f32", "kind": "norm_grad", "rows": 4099, "width": 1001, "dtype": "f32", "param": "f32", "residual": False, "p": 0.0,
         "bound": False},
        # the training batch's gradients
        {"name": "norm_grad_16k_bf16", "kind": "norm_grad", "rows": 16384, "width": 4096, "dtype": "bf16", "param": "f32", "residual": True, "p": 0.1,
         "bound": True},
        # a short odd sequence of a small model
        {"name": "dropout_37_f16", "kind": "dropout", "rows": 37, "width": 1408, "dtype": "f16", "residual": False, "p": 0.2, "bound": True},
        # a training batch's, added to the residual
        {"name": "dropout_16k_bf16", "kind": "dropout", "rows": 16384, "width": 4096, "dtype": "bf16", "residual": True, "p": 0.1, "bound": False},
        # the loss of a small batch
        {"name": "balance_48_f32", "kind": "balance", "tokens": 48, "experts": 64, "k": 6, "dtype": "f32", "renormalize": True, "masked": False,
         "grad": False, "bound": True},
        # a training batch of odd length with forbidden experts and padding tokens, forward and backward
        {"name": "balance_32k_bf16_grad", "kind": "balance", "tokens": 32771, "experts": 256, "k": 8, "dtype": "bf16", "renormalize": False,
         "masked": True, "grad": True, "bound": False},
        # one token of one request
        {"name": "adapted_1_f16", "kind": "adapted", "tokens": 1, "requests": 1, "adapters": 64, "rank": 16, "n": 4096, "kdim": 2048, "dtype": "f16",
         "bare": 0.0, "bound": True},
        # a decoding batch: a token of each request, most with an adapter of their own
        {"name": "adapted_48_bf16", "kind": "adapted", "tokens": 48, "requests": 48, "adapters": 64, "rank": 16, "n": 4096, "kdim": 4096,
         "dtype": "bf16", "bare": 0.1, "bound": True},
        # prompts of odd lengths beside decoding requests
        {"name": "adapted_1k_f16", "kind": "adapted", "tokens": 1031, "requests": 40, "adapters": 96, "rank": 8, "n": 1000, "kdim": 1416, "dtype": "f16",
         "bare": 0.2, "bound": False},
        # a batch of prompts
        {"name": "adapted_8k_bf16", "kind": "adapted", "tokens": 8192, "requests": 12, "adapters": 32, "rank": 64, "n": 4096, "kdim": 4096,
         "dtype": "bf16", "bare": 0.1, "bound": False},
    ]


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "dropout", "balance", "adapted", "adapted"])
    case = {"kind": kind, "bound": rng.random() < 0.5}
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("norm", "norm_grad", "dropout"):
        while True:
            rows, width = _log_size(rng, 1, 40000), _log_size(rng, 8, 16384)
            if rng.random() < 0.7:
                width = (width + 7) // 8 * 8
            if rows * width * BYTES[dtype] <= 134_217_728:
                break
        p = rng.choice([0.0, 0.1, 0.25, 0.5])
        if kind == "dropout":
            p = p or 0.1
        case.update(rows=rows, width=width, dtype=dtype, residual=rng.random() < 0.5, p=p)
        if kind != "dropout":
            case.update(param=rng.choice(["f32", dtype]))
    elif kind == "balance":
        experts = rng.choice([8, 16, 40, 60, 64, 128, 160, 256, 384])
        case.update(tokens=_log_size(rng, 1, 32771), experts=experts, k=rng.randint(1, 8), dtype=dtype, renormalize=rng.random() < 0.5,
                    masked=rng.random() < 0.5, grad=rng.random() < 0.5)
    else:
        while True:
            tokens, rank = _log_size(rng, 1, 12000), rng.choice([8, 16, 16, 32, 64, 128])
            n, kdim, adapters = max(64, _log_size(rng, 128, 6000) // 8 * 8), max(64, _log_size(rng, 128, 6000) // 8 * 8), _log_size(rng, 1, 200)
            if tokens * n * kdim <= 8192 * 4096 * 4096 and adapters * rank * (n + kdim) <= 1 << 28:
                break
        case.update(tokens=tokens, requests=min(tokens, _log_size(rng, 1, 64)), adapters=adapters, rank=rank, n=n, kdim=kdim,
                    dtype=rng.choice(["bf16", "f16"]), bare=rng.choice([0.0, 0.1, 0.5]))
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------

def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + salt)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _stream(g, rows, width, dtype):
    """Rows of a residual stream: features have offsets and scales of their own."""
    scale = torch.exp(torch.randn(width, generator=g, device="cuda") * 0.5)
    offset = torch.randn(width, generator=g, device="cuda") * 0.5 + 0.3
    out = torch.empty((rows, width), dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // width)
    for at in range(0, rows, step):
        part = out[at:at + step]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(scale).add_(offset))
    return out


def _request_lengths(case):
    """Tokens of each request: one at least, a few requests have most of them."""
    r = np.random.default_rng([case["tokens"], case["requests"]])
    share = np.exp(r.normal(0.0, 1.5, case["requests"]))
    lengths = 1 + np.floor(share / share.sum() * (case["tokens"] - case["requests"])).astype(np.int64)
    lengths[np.argmax(lengths)] += case["tokens"] - int(lengths.sum())
    return lengths


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind in ("norm", "norm_grad", "dropout"):
        rows, width = case["rows"], case["width"]
        if case["p"] > 0:                                     # a seed and an offset that a training loop raises every step
            state["seed"] = torch.stack([torch.randint(-(1 << 62), 1 << 62, (), generator=g, device="cuda"),
                                         torch.randint(0, 1 << 34, (), generator=g, device="cuda")])
        if kind == "dropout":
            state["x"] = _normal(g, (rows, width), dtype)
            state["residual"] = _stream(g, rows, width, dtype) if case["residual"] else None
        else:
            param = DTYPES[case["param"]]
            state["weight"] = (torch.randn(width, generator=g, device="cuda") * 0.2 + 1.0).to(param)
            state["bias"] = (torch.randn(width, generator=g, device="cuda") * 0.2).to(param)
            state["x"] = _stream(g, rows, width, dtype)
            if kind == "norm":
                state["residual"] = _stream(g, rows, width, dtype) if case["residual"] else None
            else:                                             # x: what was normalised, with its statistics of the forward pass
                var, mean = torch.var_mean(state["x"].float(), dim=1, correction=0)
                state["mean"], state["rstd"] = mean, torch.rsqrt(var + EPS)
                state["dy"] = _normal(g, (rows, width), dtype, 0.1)
                state["dsum"] = _normal(g, (rows, width), dtype, 0.1) if case["residual"] else None
    elif kind == "balance":
        tokens, experts, k = case["tokens"], case["experts"], case["k"]
        liked = torch.randn(experts, generator=g, device="cuda") * 0.5
        logits = (torch.randn((tokens, experts), generator=g, device="cuda") + liked).to(dtype)
        if case["masked"]:
            off = torch.rand((tokens, experts), generator=g, device="cuda") < 0.05
            off |= torch.rand((tokens, 1), generator=g, device="cuda") < 0.02          # a padding token: no expert at all
            logits.masked_fill_(off, float("-inf"))
        top = torch.sort(logits.float(), dim=1, descending=True, stable=True)
        ids, chosen = top.indices[:, :k], top.values[:, :k] > float("-inf")
        base = torch.where(top.values[:, :1] > float("-inf"), top.values[:, :1], torch.zeros_like(top.values[:, :1]))
        e = torch.exp(logits.float() - base)
        over = torch.gather(e, 1, ids).sum(1, keepdim=True) if case["renormalize"] else e.sum(1, keepdim=True)
        weights = torch.gather(e, 1, ids) / torch.where(over > 0, over, torch.ones_like(over))
        key, order = torch.sort(torch.where(chosen, ids, torch.full_like(ids, experts)).reshape(-1), stable=True)
        offsets = torch.searchsorted(key, torch.arange(experts + 1, device="cuda")).to(torch.int32)
        slots = torch.empty_like(order)
        slots[order] = torch.arange(order.numel(), device="cuda")
        none = torch.full_like(order, -1)
        state.update(logits=logits, weights=weights.contiguous(), experts=torch.where(chosen, ids, torch.full_like(ids, -1)).to(torch.int32),
                     offsets=offsets, rows=torch.where(key < experts, order // k, none).to(torch.int32),
                     slots=torch.where(chosen.reshape(-1), slots, none).view(tokens, k).to(torch.int32))
        if case["grad"]:
            state["dloss"] = torch.full((), 0.01, device="cuda")
            state["dweights"] = torch.randn((tokens, k), generator=g, device="cuda") * 1e-3
    else:
        tokens, adapters, rank, n, kdim = (case[s] for s in ("tokens", "adapters", "rank", "n", "kdim"))
        r = np.random.default_rng([seed, tokens, adapters])
        of_request = r.integers(0, adapters, case["requests"])
        of_request[r.random(case["requests"]) < case["bare"]] = -1
        ids = np.repeat(of_request, _request_lengths(case)).astype(np.int32)
        state.update(x=_normal(g, (tokens, kdim), dtype), weight=_normal(g, (n, kdim), dtype, kdim ** -0.5),
                     a=_normal(g, (adapters, rank, kdim), dtype, kdim ** -0.5), b=_normal(g, (adapters, n, rank), dtype, 0.1),
                     scale=torch.rand(adapters, generator=g, device="cuda") * 0.5 + 0.5, ids=torch.from_numpy(ids).cuda())
        used = np.unique(ids[ids >= 0])
        state["tokens_of"] = [(int(i), torch.from_numpy(np.flatnonzero(ids == i)).cuda()) for i in used]
    if own:
        state["pass"] = _own_pass(state)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return state["pass"]() if own else _run_plain(state)


def _own_pass(state):
    """The framework's calls of one pass.  ``bound``: a serving or training loop over fixed buffers, which binds its arguments once and
    launches every step; otherwise the plain calls, which check their arguments and allocate their outputs."""
    from flexspmv_b200 import adapters, experts, residual
    case = state["case"]
    kind = case["kind"]

    def call(op, *args, **kwargs):
        return experts.bind(op, *args, **kwargs).launch if case["bound"] else lambda: op(*args, **kwargs)

    if kind == "norm":
        norm = call(residual.layer_norm, state["x"], state["weight"], state["bias"], eps=EPS, residual=state["residual"], p=case["p"],
                    seed=state.get("seed"))

        def forward():
            out = norm()
            named = {"y": out.y, "mean": out.mean, "rstd": out.rstd}
            if out.sum is not None:
                named["sum"] = out.sum
            return named
        return forward
    if kind == "norm_grad":
        grad = call(residual.layer_norm_backward, state["dy"], state["x"], state["weight"], state["mean"], state["rstd"], dsum=state["dsum"],
                    p=case["p"], seed=state.get("seed"))

        def backward():
            out = grad()
            return {"dx": out.dx, "dresidual": out.dresidual, "dweight": out.dweight, "dbias": out.dbias}
        return backward
    if kind == "dropout":
        drop = call(residual.dropout, state["x"], case["p"], state["seed"], residual=state["residual"])
        return lambda: {"out": drop()}
    if kind == "balance":
        plan = experts.Plan(state["weights"], state["experts"], state["offsets"], state["rows"], state["slots"], case["renormalize"])
        loss = call(experts.balance_loss, state["logits"], plan)

        def balance():
            b = loss()
            out = {"loss": b.loss, "counts": b.counts, "mean": b.mean}
            if case["grad"]:
                out["dlogits"] = experts.balance_loss_backward(state["dloss"], state["logits"], b, plan=plan, dweights=state["dweights"])
            return out
        return balance
    # a batch's plan serves all of a model's projections
    plan = adapters.plan(state["ids"], case["adapters"])
    y = call(adapters.project, state["x"], state["weight"], state["a"], state["b"], plan, scale=state["scale"])
    return lambda: {"y": y()}


def _run_plain(state):
    case = state["case"]
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "dropout": _plain_dropout, "balance": _plain_balance,
            "adapted": _plain_adapted}[case["kind"]](state, case)


_WORD = 0xFFFFFFFF


def _plain_random(rows, width, seed):
    """Random words of a matrix's values, as whole numbers of 64 bits (products that pass 63 wrap, and their words are what they are)."""
    groups = (width + 3) // 4
    c0 = torch.arange(groups, device="cuda").repeat(rows)
    c1 = torch.arange(rows, device="cuda").repeat_interleave(groups)
    c2 = (seed[1] & _WORD).expand_as(c0)
    c3 = ((seed[1] >> 32) & _WORD).expand_as(c0)
    k0, k1 = seed[0] & _WORD, (seed[0] >> 32) & _WORD
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _WORD) ^ c1 ^ k0, b & _WORD, ((a >> 32) & _WORD) ^ c3 ^ k1, a & _WORD
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    return torch.stack([c0, c1, c2, c3], dim=1).view(rows, groups * 4)[:, :width]


def _plain_drop(x, p, seed):
    if p == 0.0:
        return x
    keep = _plain_random(x.shape[0], x.shape[1], seed) >= int(p * 2.0 ** 32)
    return torch.where(keep, x * (1.0 / (1.0 - p)), torch.zeros_like(x))


def _plain_norm(state, case):
    x, residual = state["x"], state["residual"]
    s = _plain_drop(x.float(), case["p"], state.get("seed"))
    if residual is not None:
        s = residual.float() + s
    mean = s.mean(dim=1, keepdim=True)
    centred = s - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    y = centred * rstd * state["weight"].float() + state["bias"].float()
    out = {"y": y.to(x.dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if residual is not None or case["p"] > 0:
        out["sum"] = s.to(x.dtype)
    return out


def _plain_norm_grad(state, case):
    dtype, param = state["x"].dtype, state["weight"].dtype
    dy, rstd = state["dy"].float(), state["rstd"][:, None]
    normed = (state["x"].float() - state["mean"][:, None]) * rstd
    g = dy * state["weight"].float()
    ds = rstd * (g - g.mean(dim=1, keepdim=True) - normed * (g * normed).mean(dim=1, keepdim=True))
    if state["dsum"] is not None:
        ds = ds + state["dsum"].float()
    return {"dx": _plain_drop(ds, case["p"], state.get("seed")).to(dtype), "dresidual": ds.to(dtype), "dweight": (dy * normed).sum(dim=0).to(param),
            "dbias": dy.sum(dim=0).to(param)}


def _plain_dropout(state, case):
    out = _plain_drop(state["x"].float(), case["p"], state["seed"])
    if state["residual"] is not None:
        out = state["residual"].float() + out
    return {"out": out.to(state["x"].dtype)}


def _plain_balance(state, case):
    logits = state["logits"]
    l = logits.float()
    experts = l.shape[1]
    counts = state["offsets"][1:] - state["offsets"][:-1]
    top = l.max(dim=1, keepdim=True).values
    there = top > float("-inf")
    e = torch.exp(l - torch.where(there, top, torch.zeros_like(top)))
    total = e.sum(dim=1, keepdim=True)
    p = e / torch.where(there, total, torch.ones_like(total))
    tokens = there.sum().clamp(min=1).float()
    pairs = counts.sum().clamp(min=1).float()
    mean = p.sum(dim=0) / tokens
    out = {"loss": (counts.float() * mean).sum() * experts / pairs, "counts": counts, "mean": mean}
    if case["grad"]:
        c = counts.float()
        scale = state["dloss"] * experts / (pairs * tokens)
        dl = scale * p * (c - (p * c).sum(dim=1, keepdim=True))
        ids = state["experts"].long()
        chosen, at, w = ids >= 0, ids.clamp(min=0), state["weights"]
        dw = torch.where(chosen, state["dweights"], torch.zeros_like(w))
        middle = (dw * w).sum(dim=1, keepdim=True)
        if case["renormalize"]:
            dl = dl.scatter_add(1, at, torch.where(chosen, w * (dw - middle), torch.zeros_like(w)))
        else:
            dl = dl + p * (torch.zeros_like(l).scatter_add_(1, at, dw) - middle)
        out["dlogits"] = dl.to(logits.dtype)
    return out


def _plain_adapted(state, case):
    x = state["x"].float()
    y = x @ state["weight"].float().t()
    for i, tokens in state["tokens_of"]:
        h = x[tokens] @ state["a"][i].float().t() * state["scale"][i]
        y[tokens] += h @ state["b"][i].float().t()
    return {"y": y.to(state["x"].dtype)}


# ---- cost and definition ------------------------------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; adapters that no token has are not read."""
    kind, b = case["kind"], BYTES[case["dtype"]]
    if kind in ("norm", "norm_grad", "dropout"):
        rows, width = case["rows"], case["width"]
        size, params = rows * width * b, width * BYTES[case.get("param", "f32")]
        random = 10 * rows * width if case["p"] > 0 else 0            # whole-number operations of the generator
        if kind == "dropout":
            return {"bytes": size * (2 + case["residual"]), "flops": 2 * rows * width + random}
        if kind == "norm":
            arrays = 2 + case["residual"] + (case["residual"] or case["p"] > 0)
            return {"bytes": size * arrays + 2 * params + 8 * rows, "flops": 8 * rows * width + random}
        return {"bytes": size * (3 + case["residual"] + (case["p"] > 0)) + 3 * params + 8 * rows, "flops": 14 * rows * width + random}
    if kind == "balance":
        te, tk = case["tokens"] * case["experts"], case["tokens"] * case["k"]
        nbytes = te * b + case["experts"] * 12
        if case["grad"]:
            nbytes += te * b + tk * 12
        return {"bytes": nbytes, "flops": te * (12 if case["grad"] else 4)}
    tokens, rank, n, kdim = case["tokens"], case["rank"], case["n"], case["kdim"]
    # of a uniform choice for each request
    used = case["adapters"] * (1.0 - (1.0 - 1.0 / case["adapters"]) ** (case["requests"] * (1.0 - case["bare"])))
    nbytes = (n * kdim + tokens * (n + kdim)) * b + used * rank * (n + kdim) * b + tokens * 4
    return {"bytes": int(nbytes), "flops": int(2 * tokens * (n * kdim + (1.0 - case["bare"]) * rank * (n + kdim)))}


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "norm_grad": _exact_norm_grad, "dropout": _exact_dropout, "balance": _exact_balance,
            "adapted": _exact_adapted}[case["kind"]](state, case)


def _exact_keep(rows, width, p, seed):
    """Which values are kept, in whole numbers on the host, some rows at a time."""
    seed, offset = (int(v) & (1 << 64) - 1 for v in seed.tolist())
    groups = (width + 3) // 4
    keep = np.empty((rows, width), dtype=bool)
    step = max(1, (1 << 18) // groups)
    m0, m1, low, half = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(_WORD), np.uint64(32)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        c = np.empty((4, n, groups), dtype=np.uint64)
        c[0], c[1] = np.arange(groups, dtype=np.uint64)[None, :], np.arange(at, at + n, dtype=np.uint64)[:, None]
        c[2], c[3] = np.uint64(offset & _WORD), np.uint64(offset >> 32)
        key = [seed & _WORD, seed >> 32]
        for _ in range(10):
            first, second = c[0] * m0, c[2] * m1
            c = np.stack([second >> half ^ c[1] ^ np.uint64(key[0]), second & low, first >> half ^ c[3] ^ np.uint64(key[1]), first & low])
            key = [(key[0] + 0x9E3779B9) & _WORD, (key[1] + 0xBB67AE85) & _WORD]
        keep[at:at + n] = (np.moveaxis(c, 0, 2).reshape(n, groups * 4)[:, :width] >= np.uint64(math.floor(p * 2 ** 32)))
    return torch.from_numpy(keep).cuda()


def _exact_drop(x, state, case):
    if case["p"] == 0.0:
        return x
    return x.mul_(_exact_keep(case["rows"], case["width"], case["p"], state["seed"])).div_(1.0 - case["p"])


def _exact_norm(state, case):
    s = _exact_drop(state["x"].double(), state, case)
    if state["residual"] is not None:
        s += state["residual"].double()
    var, mean = torch.var_mean(s, dim=1, correction=0, keepdim=True)
    rstd = (var + EPS) ** -0.5
    out = {"y": torch.addcmul(state["bias"].double(), (s - mean) * rstd, state["weight"].double()).cpu(), "mean": mean[:, 0].cpu(),
           "rstd": rstd[:, 0].cpu()}
    if state["residual"] is not None or case["p"] > 0:
        out["sum"] = s.cpu()
    return out


def _exact_norm_grad(state, case):
    dy, rstd = state["dy"].double(), state["rstd"].double()[:, None]
    normed = state["x"].double().sub_(state["mean"].double()[:, None]).mul_(rstd)
    out = {"dweight": torch.einsum("rc,rc->c", dy, normed).cpu(), "dbias": dy.sum(0).cpu()}
    g = dy.mul_(state["weight"].double())
    width = case["width"]
    first, second = g.sum(1, keepdim=True) / width, torch.einsum("rc,rc->r", g, normed)[:, None] / width
    ds = g.sub_(first).sub_(normed.mul_(second)).mul_(rstd)
    if state["dsum"] is not None:
        ds += state["dsum"].double()
    out["dresidual"] = ds.cpu()
    out["dx"] = _exact_drop(ds, state, case).cpu()
    return {name: out[name] for name in ("dx", "dresidual", "dweight", "dbias")}


def _exact_dropout(state, case):
    out = _exact_drop(state["x"].double(), state, case)
    if state["residual"] is not None:
        out += state["residual"].double()
    return {"out": out.cpu()}


def _exact_balance(state, case):
    l = state["logits"].double().cpu().numpy()
    tokens, experts = l.shape
    ids = state["experts"].cpu().numpy()
    counts = np.bincount(ids[ids >= 0], minlength=experts)
    there = np.isfinite(l).any(axis=1)
    p = np.zeros_like(l)
    e = np.exp(l[there] - l[there].max(axis=1, keepdims=True))
    p[there] = e / e.sum(axis=1, keepdims=True)
    n, pairs = max(1, int(there.sum())), max(1, int(counts.sum()))
    mean = p.sum(axis=0) / n
    out = {"loss": torch.tensor(float(mean @ counts) * experts / pairs, dtype=torch.float64), "counts": torch.from_numpy(counts.astype(np.int32)),
           "mean": torch.from_numpy(mean)}
    if case["grad"]:
        dl = float(state["dloss"].double()) * experts / (pairs * n) * p * (counts - (p @ counts)[:, None])
        ok, w = ids >= 0, state["weights"].double().cpu().numpy()
        g = np.where(ok, state["dweights"].double().cpu().numpy(), 0.0)
        rest = (g * w).sum(axis=1, keepdims=True)
        token, choice = np.nonzero(ok)
        if case["renormalize"]:
            np.add.at(dl, (token, ids[token, choice]), (w * (g - rest))[token, choice])
        else:
            np.add.at(dl, (token, ids[token, choice]), g[token, choice] * p[token, ids[token, choice]])
            dl -= p * rest
        out["dlogits"] = torch.from_numpy(dl)
    return out


def _exact_adapted(state, case):
    x = state["x"].double()
    y = torch.einsum("tk,nk->tn", x, state["weight"].double())
    ids = state["ids"].long()
    for i in torch.unique(ids).tolist():
        if i >= 0:
            t = torch.nonzero(ids == i).view(-1)
            h = torch.einsum("tk,rk->tr", x[t], state["a"][i].double())
            y.index_add_(0, t, torch.einsum("tr,nr->tn", h, state["b"][i].double()) * state["scale"][i].double())
    return {"y": y.cpu()}
