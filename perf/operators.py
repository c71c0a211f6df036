"""Timed cases of the mixture-of-experts operators: the router with its losses, the moves of rows into
expert order and back, and the product with 4-bit expert weights.

`own = False` computes each in a plain form of elementary torch operations in 32 bits; `own = True`
calls the framework. Sizes are those of the framework's mixture-of-experts workloads (64 or 8 experts,
16384 routed rows, N 14336, K 4096) and generic ones around them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


def listed():
    return [
        # one decoding step of a few sequences: latency alone counts
        _route("route-decode", tokens=4, experts=64, top_k=2, dtype="f16"),
        # a short padded batch, an expert count that is no power of two, two experts switched off
        _route("route-odd-train", tokens=999, experts=37, top_k=5, dtype="bf16", normalize=False, masked=0.1,
               closed=2, train=True),
        # the router of the 64-expert layer over a training batch
        _route("route-layer-train", tokens=16384, experts=64, top_k=2, dtype="f32", train=True),
        # many fine-grained experts over a long-context batch with padding
        _route("route-large-train", tokens=131072, experts=256, top_k=8, dtype="f32", masked=0.05, train=True),
        # rows of one decoding step
        _rows("rows-decode", tokens=4, top_k=2, width=4096, dtype="f16"),
        # an odd width (no row is aligned) and slots that went to no expert
        _rows("rows-odd-train", tokens=777, top_k=3, width=257, dtype="f32", unrouted=0.1, train=True),
        # the 16384 routed rows of the 64-expert layer, both directions
        _rows("rows-layer-train", tokens=8192, top_k=2, width=4096, dtype="bf16", train=True),
        # fine-grained experts at serving: many rows a token, FP32 results of the down-projection combined
        _rows("rows-fine-serve", tokens=4096, top_k=8, width=2048, dtype="f32"),
        # one token through one weight matrix: a matrix-vector product
        _q4("q4-token", experts=1, active=1, rows=1, n=4096, k=4096, group=128, dtype="f16", out="f16"),
        # one token, two of eight experts, up-projection with its activation
        _q4("q4-moe-token", experts=8, active=2, rows=2, n=14336, k=4096, group=128, dtype="bf16", out="bf16",
            bias=True, act="gelu", gather=True),
        # odd sizes, partial last group, zero points
        _q4("q4-odd", experts=5, active=3, rows=19, n=385, k=257, group=32, dtype="bf16", out="f32", zeros=True,
            bias=True, act="relu"),
        # a decoding batch that reaches every expert, down-projection
        _q4("q4-moe-batch", experts=8, active=8, rows=64, n=4096, k=14336, group=64, dtype="f16", out="f32",
            zeros=True),
    ]


def _route(name, tokens, experts, top_k, dtype, normalize=True, masked=0.0, closed=0, train=False):
    return dict(name=name, op="route", tokens=tokens, experts=experts, top_k=top_k, dtype=dtype, normalize=normalize,
                masked=masked, closed=closed, train=train)


def _rows(name, tokens, top_k, width, dtype, unrouted=0.0, train=False):
    return dict(name=name, op="rows", tokens=tokens, top_k=top_k, width=width, dtype=dtype, unrouted=unrouted,
                train=train)


def _q4(name, experts, active, rows, n, k, group, dtype, out, zeros=False, bias=False, act="none", gather=False):
    return dict(name=name, op="q4", experts=experts, active=active, rows=rows, n=n, k=k, group=group, dtype=dtype,
                out=out, zeros=zeros, bias=bias, act=act, gather=gather)


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi; half of the time a multiple of a power of two."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 1 << max(0, v.bit_length() - 3)
        v = v // step * step
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["route", "rows", "q4"])
    most = [max(work(c)[what] for c in listed() if c["op"] == op) for what in ("bytes", "flops")]
    while True:
        c = _drawn(rng, op)
        if work(c)["bytes"] <= most[0] and work(c)["flops"] <= most[1]:
            return c


def _drawn(rng, op):
    if op == "route":
        experts = _spread(rng, 8, 256)
        c = _route("", tokens=_spread(rng, 1, 131072), experts=experts, top_k=rng.randint(1, 8),
                   dtype=rng.choice(list(DTYPES)), normalize=rng.random() < 0.6, masked=rng.choice([0.0, 0.05, 0.4]),
                   closed=rng.choice([0, 0, 1, min(experts - 1, 5)]), train=rng.random() < 0.6)
    elif op == "rows":
        top_k = rng.randint(1, 8)
        width = _spread(rng, 64, 8192)
        c = _rows("", tokens=_spread(rng, 1, 65536), top_k=top_k, width=width, dtype=rng.choice(list(DTYPES)),
                  unrouted=rng.choice([0.0, 0.0, 0.2]), train=rng.random() < 0.6)
    else:
        most = 8 * 14336 * 4096
        n, k = _spread(rng, 64, 14336), _spread(rng, 64, 14336)
        experts = rng.randint(1, max(1, min(64, most // (n * k))))
        active = rng.randint(1, min(experts, 8))
        dtype = rng.choice(["f16", "bf16"])
        c = _q4("", experts=experts, active=active, rows=active + rng.choice([0, rng.randint(0, 64 - active)]), n=n,
                k=k, group=rng.choice([32, 64, 128]), dtype=dtype, out=rng.choice(["f32", dtype]),
                zeros=rng.random() < 0.4, bias=rng.random() < 0.4, act=rng.choice(["none", "relu", "gelu"]),
                gather=rng.random() < 0.4)
    del c["name"]
    return c


def work(case):
    c = case
    if c["op"] == "route":
        s = 4 if c["dtype"] == "f32" else 2
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        # logits and mask in; indices, weights, positions and row tokens, lse, per-expert results out
        nbytes = t * e * s + t + t * k * 16 + t * 4 + e * 8
        flops = t * e * 8
        if c["train"]:  # the gradient of the weights in, the gradient of the logits out
            nbytes += t * k * 4 + t * e * s
            flops += t * e * 8
        return {"bytes": nbytes, "flops": flops}
    if c["op"] == "rows":
        s = 4 if c["dtype"] == "f32" else 2
        slots = c["tokens"] * c["top_k"]
        row = c["width"] * s
        # dispatch: x in, packed out; combine: packed in, out; positions and weights
        nbytes = c["tokens"] * row * 2 + slots * row * 2 + slots * 8
        flops = 2 * slots * c["width"]
        if c["train"]:  # combine's gradient: grad_out in, grad_packed out; dispatch's: packed in, grad_x out
            nbytes += c["tokens"] * row * 2 + slots * row * 2 + slots * 4
            flops += 4 * slots * c["width"]
        return {"bytes": nbytes, "flops": flops}
    n, k, g = c["n"], c["k"], -(-c["k"] // c["group"])
    weights = n * ((k + 1) // 2) + n * g * (3 if c["zeros"] else 2) + (4 * n if c["bias"] else 0)
    tokens = _tokens(c)
    nbytes = c["active"] * weights + tokens * k * 2 + c["rows"] * n * (4 if c["out"] == "f32" else 2)
    return {"bytes": nbytes, "flops": 2 * c["rows"] * n * k}


def _tokens(c):
    """Rows of A: fewer than the product's rows where it gathers them (a token goes to two experts)."""
    return -(-c["rows"] // 2) if c["gather"] else c["rows"]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = {"case": c}
    dt = DTYPES[c["dtype"]]

    def normal(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device=DEVICE, generator=g) * std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=DEVICE, generator=g)

    def empty(*shape, dtype=torch.float32):
        return torch.zeros(*shape, device=DEVICE, dtype=dtype)

    if c["op"] == "route":
        t, e, k = c["tokens"], c["experts"], c["top_k"]
        # some experts are liked better than others, as the balance loss finds them
        logits = normal(t, e, std=1.5) + normal(1, e, std=0.5)
        if c["closed"]:
            logits[:, torch.randperm(e, device=DEVICE, generator=g)[:c["closed"]]] = float("-inf")
        state["logits"] = logits.to(dt)
        state["mask"] = (uniform(t) >= c["masked"]).to(torch.uint8) if c["masked"] else None
        state["grad_weights"] = normal(t, k)
        state["grad_losses"] = torch.tensor([0.01, 0.001], device=DEVICE) * (0.5 + uniform(2))
        i32 = torch.int32
        state["out"] = {"indices": empty(t, k, dtype=i32), "weights": empty(t, k), "positions": empty(t, k, dtype=i32),
                        "rows": empty(e, dtype=i32), "row_tokens": empty(t * k, dtype=i32), "losses": empty(3),
                        "lse": empty(t), "prob_mean": empty(e)}
        if c["train"]:
            state["out"]["grad_logits"] = empty(t, e, dtype=dt)
        if own:
            import grouped_gemm_gpu_kernel_b200 as gg
            state["router"] = gg.MoeRouter(e, k, t, logit_type=_type(gg, c["dtype"]), normalize=c["normalize"])
    elif c["op"] == "rows":
        t, k, w = c["tokens"], c["top_k"], c["width"]
        experts = torch.randint(0, 64, (t * k,), device=DEVICE, generator=g)
        gone = uniform(t * k) < c["unrouted"]
        order = torch.argsort(torch.where(gone, 64, experts), stable=True)
        place = torch.empty_like(order)
        place[order] = torch.arange(t * k, device=DEVICE)
        state["positions"] = torch.where(gone, -1, place).to(torch.int32).view(t, k)
        state["weights"] = torch.softmax(normal(t, k), dim=1)
        state["x"] = normal(t, w, dtype=dt)
        state["y"] = normal(t * k, w, dtype=dt)
        state["out"] = {"packed": empty(t * k, w, dtype=dt), "out": empty(t, w, dtype=dt)}
        if c["train"]:
            state["grad_out"] = normal(t, w, dtype=dt)
            state["grad_rows"] = normal(t * k, w, dtype=dt)
            state["out"] |= {"grad_packed": empty(t * k, w, dtype=dt), "grad_weights": empty(t, k),
                             "grad_x": empty(t, w, dtype=dt)}
        if own:
            import grouped_gemm_gpu_kernel_b200 as gg
            state["gg"] = gg
    else:
        e, n, k, r = c["experts"], c["n"], c["k"], c["rows"]
        groups = -(-k // c["group"])
        state["q"] = torch.randint(0, 256, (e, n, (k + 1) // 2), device=DEVICE, generator=g, dtype=torch.uint8)
        # weights of about the size 1 / sqrt(k)
        state["scales"] = ((0.5 + uniform(e, n, groups)) * (0.2 / math.sqrt(k))).to(dt)
        state["zeros"] = (torch.randint(5, 11, (e, n, groups), device=DEVICE, generator=g, dtype=torch.uint8)
                          if c["zeros"] else None)
        state["bias"] = normal(e, n, std=0.1) if c["bias"] else None
        busy = torch.randperm(e, device=DEVICE, generator=g)[:c["active"]]
        more = torch.randint(0, c["active"], (r - c["active"],), device=DEVICE, generator=g)
        chosen = torch.cat([busy, busy[more]])
        state["rows"] = torch.zeros(e, device=DEVICE, dtype=torch.int32).index_add_(
            0, chosen, torch.ones(r, device=DEVICE, dtype=torch.int32))
        tokens = _tokens(c)
        state["a"] = normal(tokens, k, dtype=dt)
        state["row_tokens"] = (torch.randint(0, tokens, (r,), device=DEVICE, generator=g, dtype=torch.int32)
                               if c["gather"] else None)
        state["d"] = empty(r, n, dtype=DTYPES[c["out"]])
        if own:
            import grouped_gemm_gpu_kernel_b200 as gg
            each = lambda t: [x.data_ptr() for x in t] if t is not None else None  # noqa: E731
            act = {"none": gg.Activation.kNone, "relu": gg.Activation.kReLU, "gelu": gg.Activation.kGELU}[c["act"]]
            state["plan"] = gg.Q4Plan(e, n, k, c["group"], each(state["q"]), (k + 1) // 2, each(state["scales"]),
                                      zero_ptrs=each(state["zeros"]), bias_ptrs=each(state["bias"]),
                                      input_type=gg.InputType.kF16 if c["dtype"] == "f16" else gg.InputType.kBF16,
                                      output_type=_type(gg, c["out"]), activation=act)
    return state


def _type(gg, name):
    return {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16}[name]


def run(state):
    c = state["case"]
    if c["op"] == "route":
        return _own_route(state) if own else _plain_route(state)
    if c["op"] == "rows":
        return _own_rows(state) if own else _plain_rows(state)
    return _own_q4(state) if own else _plain_q4(state)


# ---- the framework's calls ------------------------------------------------------------------------


def _done(status):
    if status != 0:
        raise RuntimeError(f"status {status}")


def _own_route(s):
    o, router = s["out"], s["router"]
    _done(router.run(s["logits"], o["indices"], o["weights"], o["positions"], o["rows"], o["losses"],
                     row_tokens=o["row_tokens"], lse=o["lse"], prob_mean=o["prob_mean"], token_mask=s["mask"]))
    if s["case"]["train"]:
        _done(router.backward(s["logits"], o["indices"], o["weights"], o["rows"], o["losses"], o["lse"],
                              s["grad_weights"], s["grad_losses"], o["grad_logits"]))
    return o


def _own_rows(s):
    o, gg = s["out"], s["gg"]
    _done(gg.moe_dispatch(s["x"], s["positions"], o["packed"]))
    _done(gg.moe_combine(s["y"], s["positions"], o["out"], weights=s["weights"]))
    if s["case"]["train"]:
        _done(gg.moe_combine_backward(s["grad_out"], s["y"], s["positions"], s["weights"], o["grad_packed"],
                                      o["grad_weights"]))
        _done(gg.moe_combine(s["grad_rows"], s["positions"], o["grad_x"]))
    return o


def _own_q4(s):
    _done(s["plan"].run(s["a"], s["rows"], s["d"], row_tokens=s["row_tokens"]))
    return s["d"]


# ---- the plain forms ------------------------------------------------------------------------------


def _plain_route(s):
    c = s["case"]
    e, k, neg = c["experts"], c["top_k"], float("-inf")
    real = s["logits"].float()
    t = real.shape[0]
    valid = (real != neg).any(1)
    if s["mask"] is not None:
        valid = valid & (s["mask"] != 0)
    l = torch.where(valid[:, None], real, 0.0)
    values, order = torch.sort(l, dim=1, descending=True, stable=True)
    kk = min(k, e)
    top, index = values[:, :kk], order[:, :kk]
    ok = valid[:, None] & (top != neg)
    if kk < k:  # fewer experts than slots
        top = torch.nn.functional.pad(top, (0, k - kk), value=neg)
        index = torch.nn.functional.pad(index, (0, k - kk))
        ok = torch.nn.functional.pad(ok, (0, k - kk))
    biggest = l.amax(1, keepdim=True)
    ex = torch.exp(l - biggest)
    total = ex.sum(1, keepdim=True)
    p = ex / total * valid[:, None]
    lse = (biggest + torch.log(total)).squeeze(1) * valid
    if c["normalize"]:
        w = torch.where(ok, torch.exp(top - top[:, :1]), 0.0)
        w = w / w.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        w = torch.where(ok, p.gather(1, index), 0.0)
    rows = torch.zeros(e, device=l.device, dtype=torch.int64).scatter_add_(0, index.reshape(-1), ok.reshape(-1).long())
    slots = torch.argsort(torch.where(ok, index, e).reshape(-1), stable=True)
    count = torch.arange(t * k, device=l.device)
    place = torch.empty_like(slots)
    place[slots] = count
    routed, n = rows.sum(), valid.sum().clamp(min=1)
    f = rows.float() / routed.clamp(min=1)
    prob_mean = p.sum(0) / n
    losses = torch.stack([e * (f * prob_mean).sum(), (lse * lse).sum() / n, valid.sum().float()])
    out = {"indices": torch.where(ok, index, -1).int(), "weights": w,
           "positions": torch.where(ok, place.view(t, k), -1).int(), "rows": rows.int(),
           "row_tokens": torch.where(count < routed, slots // k, -1).int(), "losses": losses, "lse": lse,
           "prob_mean": prob_mean}
    if c["train"]:
        g0, g1 = s["grad_losses"][0], s["grad_losses"][1]
        grad = p * (g0 * e / n * (f - (p * f).sum(1, keepdim=True)) + g1 * 2.0 / n * lse[:, None])
        gw = torch.where(ok, s["grad_weights"], 0.0)
        if c["normalize"]:
            part = w * (gw - (w * gw).sum(1, keepdim=True))
        else:
            part = w * gw
            grad = grad - p * part.sum(1, keepdim=True)
        out["grad_logits"] = grad.scatter_add(1, index, torch.where(ok, part, 0.0)).to(s["logits"].dtype)
    return out


def _plain_rows(s):
    c = s["case"]
    t, k, dt = c["tokens"], c["top_k"], s["x"].dtype
    ok = s["positions"] >= 0
    spare = t * k  # a row that takes what goes nowhere
    to = torch.where(ok, s["positions"], spare).long()
    at = torch.where(ok, s["positions"], 0).long()

    def scattered(v):
        rows = torch.zeros(t * k + 1, c["width"], device=v.device, dtype=dt)
        rows[to.reshape(-1)] = v.reshape(t * k, c["width"])
        return rows[:spare]

    def gathered(rows):
        return torch.where(ok[:, :, None], rows[at].float(), 0.0)

    y = gathered(s["y"])
    out = {"packed": scattered(s["x"][:, None, :].expand(t, k, c["width"])),
           "out": (y * s["weights"][:, :, None]).sum(1).to(dt)}
    if c["train"]:
        g = s["grad_out"].float()[:, None, :]
        out["grad_packed"] = scattered((g * s["weights"][:, :, None]).to(dt))
        out["grad_weights"] = (g * y).sum(2)
        out["grad_x"] = gathered(s["grad_rows"]).sum(1).to(dt)
    return out


def _plain_q4(s):
    c = s["case"]
    e, n, k, r, group = c["experts"], c["n"], c["k"], c["rows"], c["group"]
    q = torch.stack([s["q"] & 15, s["q"] >> 4], dim=3).view(e, n, -1)[:, :, :k].float()
    of = torch.arange(k, device=q.device) // group  # the group of each column
    q = (q - (s["zeros"].float()[:, :, of] if c["zeros"] else 8.0)) * s["scales"].float()[:, :, of]
    a = s["a"].float()
    if c["gather"]:
        a = a[s["row_tokens"].long()]
    row = torch.arange(r, device=q.device)
    expert = (row[:, None] >= torch.cumsum(s["rows"], 0)[None, :]).sum(1)
    spread = torch.zeros(e, r, k, device=q.device)
    spread[expert, row] = a
    d = torch.bmm(spread, q.transpose(1, 2))[expert, row]
    if c["bias"]:
        d = d + s["bias"][expert]
    if c["act"] == "relu":
        d = torch.clamp(d, min=0.0)
    elif c["act"] == "gelu":
        d = 0.5 * d * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (d + 0.044715 * d * d * d)))
    return d.to(DTYPES[c["out"]])


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "rows": _exact_rows, "q4": _exact_q4}[case["op"]](s)


def _exact_route(s):
    """The definition with torch's own differentiation of the weights and the two losses; whole numbers are left to
    the plain form."""
    c = s["case"]
    e = c["experts"]
    whole = dict.fromkeys(["indices", "positions", "rows", "row_tokens"])
    l = s["logits"].double().requires_grad_(True)
    live = l.detach().gt(float("-inf")).any(1)
    if s["mask"] is not None:
        live &= s["mask"].bool()
    at = live.nonzero().squeeze(1)
    with torch.enable_grad():
        x = l[at]
        lse = torch.logsumexp(x, 1)
        p = torch.exp(x - lse[:, None])
        # rank of each expert among its token's: by value, then by index
        order = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :c["top_k"]]
        picked = x.gather(1, order)
        there = picked.detach() > float("-inf")
        inside = torch.where(there, picked, -1e300)
        w = torch.softmax(inside, 1) if c["normalize"] else torch.where(there, p.gather(1, order), 0.0)
        share = torch.bincount(order[there], minlength=e).double()
        share = share / max(1.0, float(share.sum()))
        mean = p.sum(0) / max(1, at.numel())
        balance, z = e * (share * mean).sum(), (lse * lse).sum() / max(1, at.numel())
        weights = torch.zeros(l.shape[0], c["top_k"], device=l.device, dtype=torch.float64)
        slots = order.shape[1]
        gw = s["grad_weights"].double()[at][:, :slots]
        g = s["grad_losses"].double()
        goal = (torch.where(there, w * gw, 0.0)).sum() + g[0] * balance + g[1] * z
        grad = torch.autograd.grad(goal, l)[0] if c["train"] else None
    weights[at, :slots] = torch.where(there, w, 0.0).detach()
    full = torch.zeros(l.shape[0], device=l.device, dtype=torch.float64)
    full[at] = lse.detach()
    losses = torch.stack([balance.detach(), z.detach(), torch.tensor(float(at.numel()), device=l.device).double()])
    out = whole | {"weights": weights, "losses": losses, "lse": full, "prob_mean": mean.detach()}
    if c["train"]:
        out["grad_logits"] = torch.nan_to_num(grad, nan=0.0)  # a closed expert's is 0 times its infinity
    return out


def _exact_rows(s):
    c = s["case"]
    t, k, w = c["tokens"], c["top_k"], c["width"]
    flat = s["positions"].reshape(-1).long()
    slot = (flat >= 0).nonzero().squeeze(1)
    row, token = flat[slot], slot // k
    wts = s["weights"].reshape(-1)[slot].double()[:, None]
    zeros = lambda n: torch.zeros(n, w, device=flat.device, dtype=torch.float64)  # noqa: E731
    out = {"packed": zeros(t * k).index_copy_(0, row, s["x"].double()[token]),
           "out": zeros(t).index_add_(0, token, s["y"].double()[row] * wts)}
    if c["train"]:
        g = s["grad_out"].double()[token]
        out["grad_packed"] = zeros(t * k).index_copy_(0, row, g * wts)
        gw = torch.zeros(t * k, device=flat.device, dtype=torch.float64)
        out["grad_weights"] = gw.index_copy_(0, slot, (g * s["y"].double()[row]).sum(1)).view(t, k)
        out["grad_x"] = zeros(t).index_add_(0, token, s["grad_rows"].double()[row])
    return out


def _exact_q4(s):
    c = s["case"]
    n, k = c["n"], c["k"]
    groups = s["scales"].shape[2]
    out, first = [], 0
    for e, count in enumerate(s["rows"].tolist()):
        if count == 0:
            continue
        here = torch.arange(first, first + count, device=s["a"].device)
        first += count
        q = torch.empty(n, s["q"].shape[2] * 2, device=here.device, dtype=torch.float64)
        q[:, 0::2] = (s["q"][e] % 16).double()
        q[:, 1::2] = (s["q"][e] // 16).double()
        zero = s["zeros"][e].double() if c["zeros"] else torch.full((n, groups), 8.0, device=q.device).double()
        wide = lambda v: v.repeat_interleave(c["group"], dim=1)[:, :k]  # noqa: E731
        weight = (q[:, :k] - wide(zero)) * wide(s["scales"][e].double())
        d = s["a"][s["row_tokens"][here].long() if c["gather"] else here].double() @ weight.T
        if c["bias"]:
            d += s["bias"][e].double()
        if c["act"] == "relu":
            d = d.clamp(min=0.0)
        elif c["act"] == "gelu":
            d = d * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (d + 0.044715 * d ** 3))
        out.append(d)
    return torch.cat(out)
