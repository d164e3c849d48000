"""What the operators of a routed expert layer are measured on.

A routed layer is the framework's gather -> per-edge map -> reduce with a dense matrix as the map: an edge is a pair (token, choice),
its type is the expert that a router chose, the map is that expert's matrix, and the reduce adds a token's weighted results.

  route          softmax over the experts' logits, the k largest, and the plan: ragged offsets, slots and rows in expert order
                 (``grad``: with the gradient of the logits)
  grouped        y[i] = W[e] x[rows[i]] over ragged groups of rows, one expert's matrix each
  grouped_grad   its gradients: dx[i] = W[e]^T dy[i] and dW[e] = sum_i dy[i] x[rows[i]]^T
  combine        out[t] = sum_j w[t, j] z[slots[t, j]] (``grad``: its gradients dz and dw instead)
  clip           the norm over many gradient tensors, and the tensors scaled to a largest norm

``prepare`` makes what a program holds before the call, ``run`` makes the call: the framework's where ``own`` is true,
otherwise the same formulas in elementary operations of 32 bits.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CLIP_EPS = 1e-6


def listed():
    return [
        # a decoding step's router: eight tokens, where the launches count
        {"name": "route_8_f32", "kind": "route", "tokens": 8, "experts": 64, "k": 6, "dtype": "f32", "renormalize": True,
         "masked": False, "grad": False, "bound": True},
        # a training batch's router of odd length, forward and backward, with forbidden experts and padding tokens
        {"name": "route_32k_bf16_grad", "kind": "route", "tokens": 32771, "experts": 256, "k": 8, "dtype": "bf16",
         "renormalize": False, "masked": True, "grad": True, "bound": False},
        # one token's choices: eight matrices of 64 are read, a row each
        {"name": "grouped_1token_bf16", "kind": "grouped", "tokens": 1, "k": 8, "experts": 64, "n": 2048, "kdim": 4096,
         "dtype": "bf16", "skew": 0.0, "bound": True},
        # a batch of decoding requests: a few rows on every expert
        {"name": "grouped_decode_f16", "kind": "grouped", "tokens": 48, "k": 6, "experts": 64, "n": 1408, "kdim": 2048,
         "dtype": "f16", "skew": 0.3, "bound": True},
        # odd sizes, most rows on few experts, some experts without rows
        {"name": "grouped_ragged_f16", "kind": "grouped", "tokens": 5003, "k": 1, "experts": 40, "n": 1000, "kdim": 1416,
         "dtype": "f16", "skew": 2.0, "bound": False},
        # a prompt or a training batch through the layer's first matrix
        {"name": "grouped_prompt_bf16", "kind": "grouped", "tokens": 8192, "k": 4, "experts": 32, "n": 4096, "kdim": 2048,
         "dtype": "bf16", "skew": 0.3, "bound": False},
        # gradients of a small layer, weights' gradients kept in 32 bits
        {"name": "grouped_grad_4k_f32dw", "kind": "grouped_grad", "tokens": 2051, "k": 2, "experts": 16, "n": 1024, "kdim": 2048,
         "dtype": "bf16", "dw_dtype": "f32", "skew": 1.0, "bound": False},
        # gradients of a large one, in the weights' own type
        {"name": "grouped_grad_32k_bf16", "kind": "grouped_grad", "tokens": 8192, "k": 4, "experts": 32, "n": 4096, "kdim": 2048,
         "dtype": "bf16", "dw_dtype": "bf16", "skew": 0.3, "bound": False},
        # a decoding step's last operator
        {"name": "combine_16_bf16", "kind": "combine", "tokens": 16, "k": 8, "width": 2048, "dtype": "bf16", "grad": False, "bound": True},
        # its gradient in a training batch
        {"name": "combine_16k_bf16_grad", "kind": "combine", "tokens": 16384, "k": 4, "width": 4096, "dtype": "bf16", "grad": True, "bound": False},
        # a small model's gradients: many short tensors of odd lengths
        {"name": "clip_261_small_f32", "kind": "clip", "tensors": 261, "elements": 2_600_003, "dtype": "f32", "out_dtype": "f32",
         "max_norm": 1.0, "bound": True},
        # a large model's gradients in 16 bits, clipped into the optimizer's 32-bit buffers
        {"name": "clip_96_large_bf16", "kind": "clip", "tensors": 96, "elements": 400_000_001, "dtype": "bf16", "out_dtype": "f32",
         "max_norm": 1.0, "bound": True},
    ]


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _feature_size(rng, lo, hi):
    """A matrix side: a multiple of 8, as rows of 16-bit values that start on 16 bytes need."""
    n = max(8, _log_size(rng, lo, hi) // 8 * 8)
    return n


def draw(rng):
    kind = rng.choice(["route", "grouped", "grouped", "grouped_grad", "combine", "clip"])
    case = {"kind": kind, "bound": rng.random() < 0.5}
    if kind == "route":
        experts = rng.choice([8, 16, 40, 60, 64, 128, 160, 256, 384])
        case.update(tokens=_log_size(rng, 1, 32771), experts=experts, k=rng.randint(1, 8), dtype=rng.choice(["f32", "bf16", "f16"]),
                    renormalize=rng.random() < 0.5, masked=rng.random() < 0.5, grad=rng.random() < 0.5)
    elif kind in ("grouped", "grouped_grad"):
        while True:
            experts = rng.choice([1, 4, 8, 16, 32, 40, 64, 96])
            k = rng.randint(1, min(8, experts))
            tokens = _log_size(rng, 1 if kind == "grouped" else 32, 12000)
            n, kdim = _feature_size(rng, 128, 6000), _feature_size(rng, 128, 6000)
            if 2.0 * tokens * k * n * kdim <= 5.4e11 and experts * n * kdim <= 5.4e8 and 3072 not in (n, kdim):
                break
        case.update(tokens=tokens, k=k, experts=experts, n=n, kdim=kdim, dtype=rng.choice(["bf16", "f16"]),
                    skew=rng.choice([0.0, 0.3, 1.0, 2.0]))
        if kind == "grouped_grad":
            case.update(dw_dtype=rng.choice(["f32", case["dtype"]]))
    elif kind == "combine":
        while True:
            tokens, k, width = _log_size(rng, 1, 40000), rng.randint(1, 8), _feature_size(rng, 64, 8200)
            if tokens * (k + 1) * width <= 3.3e8 and width != 3072:
                break
        case.update(tokens=tokens, k=k, width=width, dtype=rng.choice(["bf16", "f16"]), grad=rng.random() < 0.5)
    else:
        dtype = rng.choice(["f32", "bf16", "f16"])
        case.update(tensors=_log_size(rng, 1, 700), elements=_log_size(rng, 10_000, 300_000_000), dtype=dtype,
                    out_dtype=rng.choice(["f32", dtype]), max_norm=rng.choice([0.1, 1.0, 1e6]))
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------

def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + salt)
    return g


def _normal(g, shape, dtype, scale=1.0):
    """Normal values; drawn in pieces along the first axis, so that the 32-bit draw of a large tensor is never held whole."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    if out.numel() <= 1 << 26:
        return out.copy_(torch.randn(shape, generator=g, device="cuda").mul_(scale))
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 26):
        part = flat[at:at + (1 << 26)]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(scale))
    return out


def _logits(g, tokens, experts, dtype, skew):
    """Router logits: some experts are liked more than others."""
    liked = torch.randn(experts, generator=g, device="cuda") * skew
    return (torch.randn((tokens, experts), generator=g, device="cuda") + liked).to(dtype)


def _plan(logits, k):
    """The plan of a batch, in plain operations: offsets, rows and slots in expert order."""
    tokens, experts = logits.shape
    ids = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :k].reshape(-1)
    key, order = torch.sort(ids, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device="cuda"))
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device="cuda")
    return offsets.to(torch.int32), (order // k).to(torch.int32), slots.view(tokens, k).to(torch.int32)


def _tensor_sizes(case):
    """Lengths of a model's tensors: a few large, many small, odd ones among them; the sum is about the case's."""
    r = np.random.default_rng([case["elements"], case["tensors"]])
    share = np.exp(r.normal(0.0, 2.0, case["tensors"]))
    sizes = np.maximum(1, np.floor(share / share.sum() * case["elements"])).astype(np.int64)
    sizes[np.argmax(sizes)] += max(0, case["elements"] - int(sizes.sum()))
    return [int(s) for s in sizes]


def _places(sizes):
    """Where each tensor starts in the flat buffer (on multiples of 64 elements), and the buffer's length."""
    starts, at = [], 0
    for s in sizes:
        starts.append(at)
        at += (s + 63) // 64 * 64
    return starts, at


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case}
    if kind == "route":
        tokens, experts = case["tokens"], case["experts"]
        logits = _logits(g, tokens, experts, dtype, 0.5)
        if case["masked"]:
            off = torch.rand((tokens, experts), generator=g, device="cuda") < 0.05
            off |= torch.rand((tokens, 1), generator=g, device="cuda") < 0.02          # a padding token: no expert at all
            logits.masked_fill_(off, float("-inf"))
        state["logits"] = logits
        if case["grad"]:
            state["dweights"] = torch.randn((tokens, case["k"]), generator=g, device="cuda")
    elif kind in ("grouped", "grouped_grad"):
        tokens, experts, n, kdim = case["tokens"], case["experts"], case["n"], case["kdim"]
        offsets, rows, _ = _plan(_logits(g, tokens, experts, torch.float32, case["skew"]), case["k"])
        state.update(x=_normal(g, (tokens, kdim), dtype), weight=_normal(g, (experts, n, kdim), dtype, kdim ** -0.5), offsets=offsets,
                     rows=rows, bounds=offsets.tolist())
        if kind == "grouped_grad":
            state["dy"] = _normal(g, (rows.numel(), n), dtype, 0.05)
    elif kind == "combine":
        tokens, k, width = case["tokens"], case["k"], case["width"]
        experts = 64
        logits = _logits(g, tokens, experts, torch.float32, 0.3)
        offsets, rows, slots = _plan(logits, k)
        top = torch.sort(torch.softmax(logits, dim=1), dim=1, descending=True, stable=True).values[:, :k]
        state.update(z=_normal(g, (tokens * k, width), dtype), weights=(top / top.sum(dim=1, keepdim=True)).contiguous(), offsets=offsets,
                     rows=rows, slots=slots)
        if case["grad"]:
            state["dout"] = _normal(g, (tokens, width), dtype, 0.1)
    else:
        sizes = _tensor_sizes(case)
        state["grads"] = [_normal(g, (s,), dtype, 2e-3) for s in sizes]
        starts, total = _places(sizes)
        # the optimizer's flat buffer, a piece for each tensor
        state["flat"] = torch.zeros(total, dtype=DTYPES[case["out_dtype"]], device="cuda")
        state["outs"] = [state["flat"][a:a + s] for a, s in zip(starts, sizes)]
    if own:
        state["pass"] = _own_pass(state)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return state["pass"]() if own else _run_plain(state)


def _own_pass(state):
    """The framework's calls of one pass.  ``bound``: a serving or training loop over fixed buffers, which binds its arguments once and
    launches every step; otherwise the plain calls, which check their arguments and allocate their outputs."""
    from flexspmv_b200 import experts
    case = state["case"]
    kind = case["kind"]

    def call(op, *args, **kwargs):
        return experts.bind(op, *args, **kwargs).launch if case["bound"] else lambda: op(*args, **kwargs)

    if kind == "route":
        forward = call(experts.route, state["logits"], case["k"], renormalize=case["renormalize"])

        def route():
            plan = forward()
            out = {"weights": plan.weights, "experts": plan.experts, "offsets": plan.offsets, "rows": plan.rows, "slots": plan.slots}
            if case["grad"]:
                out["dlogits"] = experts.route_backward(state["dweights"], state["logits"], plan)
            return out
        return route
    if kind == "grouped":
        y = call(experts.grouped_matmul, state["x"], state["weight"], state["offsets"], rows=state["rows"])
        return lambda: {"y": y()}
    if kind == "grouped_grad":
        dx = call(experts.grouped_matmul_dx, state["dy"], state["weight"], state["offsets"])
        dw = call(experts.grouped_matmul_dw, state["dy"], state["x"], state["offsets"], rows=state["rows"], dtype=DTYPES[case["dw_dtype"]])
        return lambda: {"dx": dx(), "dw": dw()}
    if kind == "combine" and case["grad"]:
        backward = call(experts.combine_backward, state["dout"], state["z"], state["slots"], state["weights"], state["offsets"])
        return lambda: dict(zip(("dz", "dweights"), backward()))
    if kind == "combine":
        out = call(experts.combine, state["z"], state["slots"], state["weights"])
        return lambda: {"out": out()}
    clip = call(experts.clip_grad_norm, state["grads"], case["max_norm"], out=state["outs"])
    return lambda: {"norm": clip(), "flat": state["flat"]}


def _run_plain(state):
    case = state["case"]
    return {"route": _plain_route, "grouped": _plain_grouped, "grouped_grad": _plain_grouped_grad, "combine": _plain_combine,
            "clip": _plain_clip}[case["kind"]](state, case)


def _plain_route(state, case):
    logits, k = state["logits"], case["k"]
    tokens, experts = logits.shape
    l = logits.float()
    ids = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = torch.gather(l, 1, ids) > float("-inf")
    top = l.max(dim=1, keepdim=True).values
    e = torch.exp(l - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = e.sum(dim=1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    weights = torch.gather(p, 1, ids)
    if case["renormalize"]:
        part = weights.sum(dim=1, keepdim=True)
        weights = weights / torch.where(part > 0, part, torch.ones_like(part))
    key, order = torch.sort(torch.where(chosen, ids, torch.full_like(ids, experts)).reshape(-1), stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device="cuda"))
    place = torch.arange(order.numel(), device="cuda")
    none = torch.full_like(order, -1)
    used = key < experts
    slots = torch.empty_like(order)
    slots[order] = torch.where(used, place, none)
    out = {"weights": weights, "experts": torch.where(chosen, ids, torch.full_like(ids, -1)).to(torch.int32),
           "offsets": offsets.to(torch.int32), "rows": torch.where(used, order // k, none).to(torch.int32),
           "slots": slots.view(tokens, k).to(torch.int32)}
    if case["grad"]:
        dw = torch.where(chosen, state["dweights"], torch.zeros_like(weights))
        mean = (dw * weights).sum(dim=1, keepdim=True)
        if case["renormalize"]:
            dl = torch.zeros_like(l).scatter_(1, ids, weights * (dw - mean))
        else:
            dl = p * (torch.zeros_like(l).scatter_(1, ids, dw) - mean)
        out["dlogits"] = dl.to(logits.dtype)
    return out


def _plain_grouped(state, case):
    x, w, b = state["x"], state["weight"], state["bounds"]
    y = torch.zeros((state["rows"].numel(), w.shape[1]), dtype=torch.float32, device="cuda")
    rows = state["rows"].long()
    for e in range(w.shape[0]):
        if b[e + 1] > b[e]:
            y[b[e]:b[e + 1]] = x[rows[b[e]:b[e + 1]]].float() @ w[e].float().t()
    return {"y": y.to(x.dtype)}


def _plain_grouped_grad(state, case):
    x, w, dy, b = state["x"], state["weight"], state["dy"], state["bounds"]
    rows = state["rows"].long()
    dx = torch.zeros((rows.numel(), w.shape[2]), dtype=torch.float32, device="cuda")
    dw = torch.zeros(w.shape, dtype=DTYPES[case["dw_dtype"]], device="cuda")
    for e in range(w.shape[0]):
        if b[e + 1] > b[e]:
            d = dy[b[e]:b[e + 1]].float()
            dx[b[e]:b[e + 1]] = d @ w[e].float()
            dw[e] = (d.t() @ x[rows[b[e]:b[e + 1]]].float()).to(dw.dtype)
    return {"dx": dx.to(dy.dtype), "dw": dw}


def _plain_combine(state, case):
    z, slots, weights = state["z"], state["slots"].long(), state["weights"]
    if not case["grad"]:
        out = torch.zeros((slots.shape[0], z.shape[1]), dtype=torch.float32, device="cuda")
        for j in range(slots.shape[1]):
            out += weights[:, j:j + 1] * z[slots[:, j]].float()
        return {"out": out.to(z.dtype)}
    dout = state["dout"].float()
    dz = torch.zeros_like(z)
    dweights = torch.empty_like(weights)
    for j in range(slots.shape[1]):
        dz[slots[:, j]] = (weights[:, j:j + 1] * dout).to(z.dtype)
        dweights[:, j] = (dout * z[slots[:, j]].float()).sum(dim=1)
    return {"dz": dz, "dweights": dweights}


def _plain_clip(state, case):
    total = torch.stack([(t.float() * t.float()).sum() for t in state["grads"]]).sum()
    norm = torch.sqrt(total)
    scale = torch.clamp(case["max_norm"] / (norm + CLIP_EPS), max=1.0)
    for t, o in zip(state["grads"], state["outs"]):
        o.copy_(t.float() * scale)
    return {"norm": norm, "flat": state["flat"]}


# ---- cost and definition ------------------------------------------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; matrices of experts without rows are not read (about: by the mean of a
    uniform choice)."""
    kind, b = case["kind"], BYTES[case["dtype"]]
    if kind == "route":
        te, tk = case["tokens"] * case["experts"], case["tokens"] * case["k"]
        nbytes = te * b + tk * 16 + (case["experts"] + 1) * 4
        if case["grad"]:
            nbytes += tk * 4 + te * b
        return {"bytes": nbytes, "flops": te * (8 if case["grad"] else 4)}
    if kind in ("grouped", "grouped_grad"):
        rows, nk = case["tokens"] * case["k"], case["n"] * case["kdim"]
        used = min(case["experts"], rows)
        if kind == "grouped":
            return {"bytes": used * nk * b + case["tokens"] * case["kdim"] * b + rows * (case["n"] * b + 4), "flops": 2 * rows * nk}
        return {"bytes": used * nk * b + case["experts"] * nk * BYTES[case["dw_dtype"]] + case["tokens"] * case["kdim"] * b
                + rows * ((case["n"] + case["kdim"]) * b + 4), "flops": 4 * rows * nk}
    if kind == "combine":
        rows, width = case["tokens"] * case["k"], case["width"]
        nbytes = rows * (width * b + 8) + case["tokens"] * width * b
        if case["grad"]:
            nbytes += rows * (width * b + 4)
        return {"bytes": nbytes, "flops": 2 * rows * width * (2 if case["grad"] else 1)}
    return {"bytes": case["elements"] * (b + BYTES[case["out_dtype"]]), "flops": 3 * case["elements"]}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(state, case)
    if kind in ("grouped", "grouped_grad"):
        return _exact_grouped(state, case)
    if kind == "combine":
        return _exact_combine(state, case)
    sums = [float(torch.linalg.vecdot(t.double(), t.double())) for t in state["grads"]]
    norm = math.sqrt(math.fsum(sums))
    scale = min(1.0, case["max_norm"] / (norm + CLIP_EPS))
    starts, total = _places([t.numel() for t in state["grads"]])
    flat = torch.zeros(total, dtype=torch.float64)
    for t, a in zip(state["grads"], starts):
        flat[a:a + t.numel()] = (t.double() * scale).cpu()
    return {"norm": torch.tensor(norm, dtype=torch.float64), "flat": flat}


def _exact_route(state, case):
    l = state["logits"].double().cpu().numpy()
    tokens, experts = l.shape
    k = case["k"]
    ids = np.argsort(-l, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(l, ids, axis=1)
    ok = ~np.isneginf(top)
    base = np.where(np.isneginf(top[:, :1]), 0.0, top[:, :1])
    e = np.exp(l - base)
    over = np.exp(top - base).sum(axis=1, keepdims=True) if case["renormalize"] else e.sum(axis=1, keepdims=True)
    over = np.where(over == 0.0, 1.0, over)
    w = np.exp(top - base) / over
    chosen = np.where(ok, ids, -1)
    flat = chosen.reshape(-1)
    counts = np.bincount(flat[flat >= 0], minlength=experts)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    slots = np.full(flat.size, -1, dtype=np.int64)
    rows = np.full(flat.size, -1, dtype=np.int64)
    pair = np.flatnonzero(flat >= 0)
    pair = pair[np.argsort(flat[pair], kind="stable")]
    slots[pair] = np.arange(pair.size)
    rows[:pair.size] = pair // k
    out = {"weights": torch.from_numpy(w), "experts": torch.from_numpy(chosen.astype(np.int32)),
           "offsets": torch.from_numpy(offsets.astype(np.int32)), "rows": torch.from_numpy(rows.astype(np.int32)),
           "slots": torch.from_numpy(slots.reshape(tokens, k).astype(np.int32))}
    if case["grad"]:
        g = np.where(ok, state["dweights"].double().cpu().numpy(), 0.0)
        mean = (g * w).sum(axis=1, keepdims=True)
        dl = np.zeros_like(l)
        if case["renormalize"]:
            np.put_along_axis(dl, ids, w * (g - mean), axis=1)
        else:
            np.put_along_axis(dl, ids, g, axis=1)
            dl = e / over * (dl - mean)
        out["dlogits"] = torch.from_numpy(dl)
    return out


def _exact_grouped(state, case):
    rows, x, w = state["rows"].long(), state["x"], state["weight"]
    count, experts = rows.numel(), w.shape[0]
    of = torch.repeat_interleave(torch.arange(experts, device="cuda"), state["offsets"].long().diff())
    grad = case["kind"] == "grouped_grad"
    first = torch.zeros((count, w.shape[2] if grad else w.shape[1]), dtype=torch.float64, device="cuda")
    dw = torch.zeros(w.shape, dtype=torch.float64) if grad else None
    for e in range(experts):
        at = torch.nonzero(of == e).view(-1)
        if at.numel() == 0:
            continue
        we, xe = w[e].double(), x[rows[at]].double()
        if grad:
            d = state["dy"][at].double()
            first[at] = torch.einsum("rn,nk->rk", d, we)
            dw[e] = torch.einsum("rn,rk->nk", d, xe).cpu()
        else:
            first[at] = torch.einsum("rk,nk->rn", xe, we)
    return {"dx": first.cpu(), "dw": dw} if grad else {"y": first.cpu()}


def _exact_combine(state, case):
    z, slots, w = state["z"], state["slots"].long(), state["weights"].double()
    tokens, k = slots.shape
    step = 2048
    if not case["grad"]:
        return {"out": torch.cat([torch.einsum("tk,tkh->th", w[a:a + step], z[slots[a:a + step]].double()).cpu()
                                  for a in range(0, tokens, step)])}
    dz = torch.zeros(z.shape, dtype=torch.float64)
    dw = torch.zeros((tokens, k), dtype=torch.float64)
    for a in range(0, tokens, step):
        d, s = state["dout"][a:a + step].double(), slots[a:a + step]
        dz[s.reshape(-1).cpu()] = torch.einsum("tk,th->tkh", w[a:a + step], d).reshape(-1, z.shape[1]).cpu()
        dw[a:a + step] = torch.einsum("th,tkh->tk", d, z[s].double()).cpu()
    return {"dz": dz, "dweights": dw}
