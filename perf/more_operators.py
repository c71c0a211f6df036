"""Timed cases of the operators around the experts' products: the root-mean-square norm with the residual's addition
and an output in 8 bits, the product of 8-bit rows and weights with a scale for each block of 128, and the gated
feed-forward of experts with its gradient.

`own = False` computes each in a plain form of elementary torch operations in 32 bits; `own = True` calls the framework.
Sizes are those of the framework's mixture-of-experts workloads (64 or 8 experts, 16384 routed rows, N 14336, K 4096)
and generic ones around them.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn,
          "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
BLOCK = 128
EPS = 1e-6
DEVICE = "cuda"


def listed():
    return [
        # the norm of one decoding step of a few sequences, into 8 bits: latency alone counts
        _norm("norm-decode-q", rows=4, width=4096, dtype="bf16", q="e4m3"),
        # a short batch, an odd width whose rows are not aligned
        _norm("norm-odd-train", rows=777, width=1003, dtype="f32", y=True, train=True),
        # the norm before the layer's experts over a training batch
        _norm("norm-layer-train", rows=16384, width=4096, dtype="bf16", y=True, train=True),
        # a long prompt: the router's input in 16 bits and the experts' rows in 8
        _norm("norm-prompt-q", rows=32768, width=4096, dtype="bf16", y=True, q="e4m3"),
        # gate and up of 8 experts for the rows of one decoding step, 8 bits in and out
        _f8("f8-gated-decode", experts=8, rows=16, n=14336, k=4096, gated=True, act="silu", out="e4m3"),
        # the way down for a few more rows
        _f8("f8-down-serve", experts=8, rows=64, n=4096, k=14336, out="bf16"),
        # a ragged set: an expert without rows, sizes that are no multiple of anything
        _f8("f8-odd", experts=5, rows=333, n=777, k=1003, out="f32", bias=True, act="gelu", idle=1),
        # the 64-expert layer's routed rows
        _f8("f8-layer", experts=64, rows=16384, n=14336, k=4096, out="bf16"),
        # the gated block on the rows of one decoding step
        _gated("gated-decode", experts=8, rows=16, n=14336, k=4096, dtype="bf16", act="silu"),
        # a ragged training batch with an idle expert
        _gated("gated-odd-train", experts=5, rows=333, n=331, k=203, dtype="f16", act="gelu", idle=1, train=True),
        # many fine-grained experts
        _gated("gated-fine-train", experts=64, rows=32768, n=1024, k=2048, dtype="bf16", act="silu", train=True),
        # 8 experts of the layer's size
        _gated("gated-layer-train", experts=8, rows=8192, n=14336, k=4096, dtype="bf16", act="silu", train=True),
    ]


def _norm(name, rows, width, dtype, y=False, q="none", residual=True, train=False):
    return dict(name=name, op="norm", rows=rows, width=width, dtype=dtype, y=y, q=q, residual=residual, train=train)


def _f8(name, experts, rows, n, k, out, dtype="e4m3", gated=False, act="none", bias=False, idle=0):
    return dict(name=name, op="f8", experts=experts, rows=rows, n=n, k=k, out=out, dtype=dtype, gated=gated, act=act,
                bias=bias, idle=idle)


def _gated(name, experts, rows, n, k, dtype, act, idle=0, train=False):
    return dict(name=name, op="gated", experts=experts, rows=rows, n=n, k=k, dtype=dtype, act=act, idle=idle, train=train)


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi; half of the time a multiple of a power of two."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        step = 1 << max(0, v.bit_length() - 3)
        v = v // step * step
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["norm", "f8", "gated"])
    most = [max(work(c)[what] for c in listed() if c["op"] == op) for what in ("bytes", "flops")]
    while True:
        c = _drawn(rng, op)
        if work(c)["bytes"] <= most[0] and work(c)["flops"] <= most[1]:
            return c


def _drawn(rng, op):
    experts = _spread(rng, 1, 64)
    idle = rng.choice([0, 0, experts // 3])
    if op == "norm":
        train = rng.random() < 0.5
        y, q = rng.choice([(True, "none"), (False, "e4m3"), (True, "e4m3"), (False, "e5m2")])
        c = _norm("", rows=_spread(rng, 1, 65536), width=_spread(rng, 64, 16384), dtype=rng.choice(["f32", "f16", "bf16"]),
                  y=y or train, q=q, residual=rng.random() < 0.7, train=train)
    elif op == "f8":
        gated = rng.random() < 0.4
        c = _f8("", experts=experts, rows=_spread(rng, 1, 16384), n=_spread(rng, 64, 14336), k=_spread(rng, 64, 14336),
                out=rng.choice(["f32", "f16", "bf16", "e4m3", "e5m2"] if gated else ["f32", "f16", "bf16"]),
                dtype=rng.choice(["e4m3", "e4m3", "e5m2"]), gated=gated, idle=idle,
                act=rng.choice(["silu", "gelu", "relu"] if gated else ["none", "none", "relu", "gelu", "silu"]),
                bias=not gated and rng.random() < 0.4)
    else:
        c = _gated("", experts=experts, rows=_spread(rng, 1, 32768), n=_spread(rng, 64, 14336), k=_spread(rng, 64, 8192),
                   dtype=rng.choice(["f16", "bf16"]), act=rng.choice(["silu", "silu", "gelu", "relu"]), idle=idle,
                   train=rng.random() < 0.6)
    del c["name"]
    return c


def _size(name):
    return {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "e5m2": 1}[name]


def _busy(c):
    """At most so many experts have rows."""
    return max(1, min(c["experts"] - c["idle"], c["rows"]))


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    c = case
    if c["op"] == "norm":
        r, w, s = c["rows"], c["width"], _size(c["dtype"])
        nbytes = r * w * s * (1 + 2 * c["residual"] + c["y"]) + w * s + 4 * r
        if c["q"] != "none":
            nbytes += r * w + 4 * r * _blocks(w)
        flops = 5 * r * w
        if c["train"]:  # the gradients of y and of h in, the row's values again; the gradient of x out
            nbytes += r * w * s * 4 + w * s + 4 * w + 4 * r
            flops += 9 * r * w
        return {"bytes": nbytes, "flops": flops}
    e, r, n, k, b = _busy(c), c["rows"], c["n"], c["k"], c["experts"]
    if c["op"] == "f8":
        both = 2 if c["gated"] else 1
        nbytes = both * e * (n * k + 4 * _blocks(n) * _blocks(k)) + r * k + 4 * r * _blocks(k) + r * n * _size(c["out"])
        nbytes += 4 * r * _blocks(n) * (_size(c["out"]) == 1) + 4 * e * n * c["bias"] + 4 * b
        return {"bytes": nbytes, "flops": 2 * both * r * n * k}
    # x and the experts' two matrices in, h out
    nbytes = 2 * (2 * e * n * k + r * k + r * n) + 4 * b
    flops = 4 * r * n * k
    if c["train"]:  # gate and up out and in, the gradient of h in, gradients of gate, up, x and all weights out
        nbytes += 2 * (4 * r * n + r * n + 2 * r * n + 2 * e * n * k + 2 * r * k + 2 * b * n * k)
        flops += 8 * r * n * k
    return {"bytes": nbytes, "flops": flops}


# ---- what a program has in hand -------------------------------------------------------------------


def _counts(c, seed):
    """Rows of each expert: some are liked better than others, `idle` of them get none."""
    rng = random.Random(seed)
    busy = rng.sample(range(c["experts"]), _busy(c))
    liked = [math.exp(rng.gauss(0.0, 0.5)) for _ in busy]
    counts = [0] * c["experts"]
    spare = c["rows"] - len(busy)
    for e, w in zip(busy, liked):
        counts[e] = 1 + int(spare * w / sum(liked))
    for j in range(c["rows"] - sum(counts)):
        counts[busy[j % len(busy)]] += 1
    return counts


def _pitched(t, rows, cols, dtype, fill=0):
    """A rows x cols view whose rows start on 16-byte boundaries."""
    unit = 16 // torch.empty(0, dtype=dtype).element_size()
    base = torch.full((*t, rows, -(-cols // unit) * unit), fill, device=DEVICE, dtype=torch.uint8 if unit == 16 else dtype)
    return base.view(dtype)[..., :cols]


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = {"case": c}
    if own:
        import grouped_gemm_gpu_kernel_b200 as gg
        kinds = {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16,
                 "e4m3": gg.OutputType.kE4M3, "e5m2": gg.OutputType.kE5M2}
        inputs = {"f16": gg.InputType.kF16, "bf16": gg.InputType.kBF16, "e4m3": gg.InputType.kE4M3, "e5m2": gg.InputType.kE5M2}
        acts = {"none": gg.Activation.kNone, "relu": gg.Activation.kReLU, "gelu": gg.Activation.kGELU, "silu": gg.Activation.kSiLU}
    dt = DTYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEVICE, generator=g) * std

    def empty(*shape, dtype=torch.float32):
        return torch.zeros(*shape, device=DEVICE, dtype=dtype)

    if c["op"] == "norm":
        r, w = c["rows"], c["width"]
        state["x"] = normal(r, w).to(dt)
        state["residual"] = normal(r, w, std=2.0).to(dt) if c["residual"] else None
        state["weight"] = (1.0 + normal(w, std=0.2)).to(dt)
        out = {"rstd": empty(r)}
        if c["residual"]:
            out["h"] = empty(r, w, dtype=dt)
        if c["y"]:
            out["y"] = empty(r, w, dtype=dt)
        if c["q"] != "none":
            out["q"] = _pitched((), r, w, DTYPES[c["q"]])
            out["scales"] = empty(r, _blocks(w))
        if c["train"]:
            state["grad_y"], state["grad_h"] = normal(r, w).to(dt), normal(r, w).to(dt)
            out |= {"grad_x": empty(r, w, dtype=dt), "grad_weight": empty(w)}
        state["out"] = out
        if own:
            state["norm"] = gg.RmsNorm(w, dtype=kinds[c["dtype"]], weight_type=kinds[c["dtype"]], eps=EPS)
        return state

    e, r, n, k = c["experts"], c["rows"], c["n"], c["k"]
    state["counts"] = _counts(c, seed)
    state["rows"] = torch.tensor(state["counts"], device=DEVICE, dtype=torch.int32)
    if c["op"] == "f8":
        state["a"], state["a_scales"] = _pitched((), r, k, dt), empty(r, _blocks(k))
        rows = normal(r, k) * torch.exp(normal(r, 1, std=0.5))
        for j in range(_blocks(k)):  # a scale for each row and 128 columns
            part = rows[:, j * BLOCK:(j + 1) * BLOCK]
            s = part.abs().amax(1) / LARGEST[c["dtype"]]
            state["a_scales"][:, j] = s
            state["a"][:, j * BLOCK:(j + 1) * BLOCK] = (part / s[:, None]).to(dt)
        names = ["b", "up"] if c["gated"] else ["b"]
        for name in names:
            q = _pitched((e,), n, k, dt)
            # weights of about the size 1 / sqrt(k), with a scale for each block of 128 x 128
            scales = (0.5 + torch.rand(e, _blocks(n), _blocks(k), device=DEVICE, generator=g)) * (4.0 / LARGEST[c["dtype"]] / math.sqrt(k))
            for j in range(e):
                q[j] = (normal(n, k).clamp(-4.0, 4.0) * (LARGEST[c["dtype"]] / 4.0)).to(dt)
            state[name], state[name + "_scales"] = q, scales
        state["bias"] = normal(e, n, std=0.1) if c["bias"] else None
        eight = _size(c["out"]) == 1
        state["d"] = _pitched((), r, n, DTYPES[c["out"]]) if eight else empty(r, n, dtype=DTYPES[c["out"]])
        state["d_scales"] = empty(r, _blocks(n)) if eight else None
        if own:
            each = lambda t: [x.data_ptr() for x in t] if t is not None else None  # noqa: E731
            state["plan"] = gg.F8Plan(e, n, k, each(state["b"]), state["b"].stride(1), each(state["b_scales"]),
                                      up_ptrs=each(state.get("up")), up_scale_ptrs=each(state.get("up_scales")),
                                      bias_ptrs=each(state["bias"]), input_type=inputs[c["dtype"]],
                                      output_type=kinds[c["out"]], activation=acts[c["act"]])
        return state

    state["x"] = _pitched((), r, k, dt)
    state["x"].copy_(normal(r, k))
    for name in ("wg", "wu"):
        state[name] = _pitched((e,), k, n, dt)
        for j in range(e):
            state[name][j] = normal(k, n, std=1.0 / math.sqrt(k)).to(dt)
    out = {"h": _pitched((), r, n, dt)}
    if c["train"]:
        state["grad_h"] = _pitched((), r, n, dt)
        state["grad_h"].copy_(normal(r, n))
        out |= {name: _pitched((), r, n, dt) for name in ("gate", "up", "grad_gate", "grad_up")}
        out["grad_x"] = _pitched((), r, k, dt)
        out |= {name: _pitched((e,), k, n, dt) for name in ("grad_wg", "grad_wu")}
    state["out"] = out
    if own:
        each = lambda t: [x.data_ptr() for x in t]  # noqa: E731
        state["plan"] = gg.GatedPlan(e, n, k, each(state["wg"]), each(state["wu"]), state["wg"].stride(1),
                                     input_type=inputs[c["dtype"]], activation=acts[c["act"]])
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "f8": _own_f8, "gated": _own_gated}[op](state)
    return {"norm": _plain_norm, "f8": _plain_f8, "gated": _plain_gated}[op](state)


# ---- the framework's calls ------------------------------------------------------------------------


def _done(status):
    if status != 0:
        raise RuntimeError(f"status {status}")


def _own_norm(s):
    o, norm = s["out"], s["norm"]
    _done(norm.run(s["x"], s["weight"], y=o.get("y"), residual=s["residual"], residual_out=o.get("h"), q=o.get("q"),
                   scales=o.get("scales"), rstd=o["rstd"]))
    if s["case"]["train"]:
        _done(norm.backward(o["h"] if "h" in o else s["x"], s["weight"], o["rstd"], s["grad_y"], o["grad_x"],
                            grad_weight=o["grad_weight"], grad_h=s["grad_h"]))
    return o


def _own_f8(s):
    _done(s["plan"].run(s["a"], s["a_scales"], s["rows"], s["d"], d_scales=s["d_scales"]))
    return {"d": s["d"]} if s["d_scales"] is None else {"d": s["d"], "scales": s["d_scales"]}


def _own_gated(s):
    o, plan = s["out"], s["plan"]
    _done(plan.run(s["x"], s["rows"], o["h"], gate=o.get("gate"), up=o.get("up")))
    if s["case"]["train"]:
        _done(plan.backward(s["x"], o["gate"], o["up"], s["grad_h"], s["rows"], o["grad_gate"], o["grad_up"],
                            grad_x=o["grad_x"], grad_gate_w=o["grad_wg"], grad_up_w=o["grad_wu"]))
    return o


# ---- the plain forms ------------------------------------------------------------------------------


def _act(x, name):
    if name == "relu":
        return torch.where(x > 0, x, 0.0)
    if name == "gelu":  # its tanh form
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    return x


def _slope(x, name):
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x))
        return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * x * x)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return p * (1.0 + x * (1.0 - p))
    return torch.ones_like(x)


def _eight_bits(y, kind):
    """(values in 8 bits, a scale for each row and 128 columns)"""
    r, w = y.shape
    pad = torch.nn.functional.pad(y, (0, _blocks(w) * BLOCK - w)).view(r, _blocks(w), BLOCK)
    scales = pad.abs().amax(2) / LARGEST[kind]
    q = pad / torch.where(scales > 0, scales, 1.0)[..., None]
    return q.clamp(-LARGEST[kind], LARGEST[kind]).reshape(r, -1)[:, :w].to(DTYPES[kind]), scales


def _plain_norm(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    out = {}
    if c["residual"]:
        out["h"] = (s["x"].float() + s["residual"].float()).to(dt)
    h = (out["h"] if c["residual"] else s["x"]).float()
    rstd = 1.0 / torch.sqrt((h * h).mean(1) + EPS)
    w = s["weight"].float()
    y = h * rstd[:, None] * w
    if c["y"]:
        out["y"] = y.to(dt)
    if c["q"] != "none":
        out["q"], out["scales"] = _eight_bits(y, c["q"])
    out["rstd"] = rstd
    if c["train"]:
        gy, xhat = s["grad_y"].float(), h * rstd[:, None]
        g = gy * w
        gx = rstd[:, None] * (g - xhat * (g * xhat).mean(1, keepdim=True)) + s["grad_h"].float()
        out["grad_x"] = gx.to(dt)
        out["grad_weight"] = (gy * xhat).sum(0)
    return out


def _wide(q, scales):
    """8-bit weights as the values they stand for."""
    n, k = q.shape
    return q.float() * scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_f8(s):
    c = s["case"]
    a = s["a"].float() * s["a_scales"].repeat_interleave(BLOCK, 1)[:, :c["k"]]
    parts, first = [], 0
    for e, count in enumerate(s["counts"]):
        if count == 0:
            continue
        rows = a[first:first + count]
        first += count
        d = rows @ _wide(s["b"][e], s["b_scales"][e]).t()
        if c["bias"]:
            d = d + s["bias"][e]
        d = _act(d, c["act"])
        if c["gated"]:
            d = d * (rows @ _wide(s["up"][e], s["up_scales"][e]).t())
        parts.append(d if _size(c["out"]) == 1 else d.to(DTYPES[c["out"]]))
    d = torch.cat(parts)
    if _size(c["out"]) > 1:
        return {"d": d}
    q, scales = _eight_bits(d, c["out"])
    return {"d": q, "scales": scales}


def _plain_gated(s):
    c = s["case"]
    dt = s["x"].dtype
    parts, first = {}, 0

    def keep(**more):
        for name, v in more.items():
            parts.setdefault(name, []).append(v.to(dt))
            # what is held in 16 bits goes on as it is held
            more[name] = parts[name][-1].float()
        return more

    for e, count in enumerate(s["counts"]):
        x = s["x"][first:first + count].float()
        here = slice(first, first + count)
        first += count
        if count == 0 and not c["train"]:
            continue
        wg, wu = s["wg"][e].float(), s["wu"][e].float()
        gate, up = x @ wg, x @ wu
        keep(h=_act(gate, c["act"]) * up)
        if c["train"]:
            v = keep(gate=gate, up=up)
            gate, up, gh = v["gate"], v["up"], s["grad_h"][here].float()
            v = keep(grad_gate=gh * up * _slope(gate, c["act"]), grad_up=gh * _act(gate, c["act"]))
            keep(grad_x=v["grad_gate"] @ wg.t() + v["grad_up"] @ wu.t(), grad_wg=x.t() @ v["grad_gate"], grad_wu=x.t() @ v["grad_up"])
    return {name: (torch.stack if name in ("grad_wg", "grad_wu") else torch.cat)(v) for name, v in parts.items()}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "f8": _exact_f8, "gated": _exact_gated}[case["op"]](s)


def _act64(x, name):
    return {"none": lambda: x, "relu": lambda: x.clamp(min=0.0), "silu": lambda: x * torch.sigmoid(x),
            "gelu": lambda: x * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3))}[name]()


def _in_groups(y, kind):
    """The nearest 8-bit values in 64 bits' reckoning, and their scales."""
    scales = torch.stack([p.abs().amax(1) for p in y.split(BLOCK, dim=1)], 1) / LARGEST[kind]
    per = scales.repeat_interleave(BLOCK, 1)[:, :y.shape[1]]
    return torch.where(per > 0, y / per, 0.0).float().to(DTYPES[kind]).double(), scales


def _exact_norm(s):
    """The definition on the stored h, the gradients by torch's own differentiation."""
    c = s["case"]
    x = s["x"].double()
    out = {}
    if c["residual"]:
        x = x + s["residual"].double()
        out["h"] = x
        x = x.float().to(s["x"].dtype).double()
    x, w = x.requires_grad_(True), s["weight"].double().requires_grad_(True)
    with torch.enable_grad():
        rstd = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
        y = x * rstd * w
        if c["train"]:
            goal = (y * s["grad_y"].double()).sum() + (x * s["grad_h"].double()).sum()
            out["grad_x"], out["grad_weight"] = torch.autograd.grad(goal, (x, w))
    y = y.detach()
    if c["y"]:
        out["y"] = y
    if c["q"] != "none":
        out["q"], out["scales"] = _in_groups(y, c["q"])
    out["rstd"] = rstd.detach().squeeze(1)
    return out


def _exact_f8(s):
    c = s["case"]
    span = lambda v, n, dim: v.double().repeat_interleave(BLOCK, dim).narrow(dim, 0, n)  # noqa: E731
    a = s["a"].double() * span(s["a_scales"], c["k"], 1)
    d = torch.empty(c["rows"], c["n"], device=a.device, dtype=torch.float64)
    ends = torch.tensor(s["counts"]).cumsum(0).tolist()
    for e, (end, count) in enumerate(zip(ends, s["counts"])):
        if not count:
            continue
        part = a[end - count:end]
        weights = [s[n][e].double() * span(span(s[n + "_scales"][e], c["n"], 0), c["k"], 1) for n in (("b", "up") if c["gated"] else ("b",))]
        got = part @ weights[0].T
        if c["bias"]:
            got += s["bias"][e].double()
        got = _act64(got, c["act"])
        d[end - count:end] = got * (part @ weights[1].T) if c["gated"] else got
    if _size(c["out"]) > 1:
        return {"d": d}
    q, scales = _in_groups(d, c["out"])
    return {"d": q, "scales": scales}


def _exact_gated(s):
    """No rounding between input and result; the gradients by torch's own differentiation, expert by expert."""
    c = s["case"]
    found = {}
    ends = torch.tensor(s["counts"]).cumsum(0).tolist()
    for e, (end, count) in enumerate(zip(ends, s["counts"])):
        x = s["x"][end - count:end].double()
        wg, wu = s["wg"][e].double(), s["wu"][e].double()
        gate, up = x @ wg, x @ wu
        if not c["train"]:
            found.setdefault("h", []).append(_act64(gate, c["act"]) * up)
            continue
        gate, up = gate.requires_grad_(True), up.requires_grad_(True)
        with torch.enable_grad():
            h = _act64(gate, c["act"]) * up
        gg_, gu = torch.autograd.grad(h, (gate, up), s["grad_h"][end - count:end].double())
        here = {"h": h.detach(), "gate": gate.detach(), "up": up.detach(), "grad_gate": gg_, "grad_up": gu,
                "grad_x": gg_ @ wg.T + gu @ wu.T, "grad_wg": x.T @ gg_, "grad_wu": x.T @ gu}
        for name, v in here.items():
            found.setdefault(name, []).append(v)
    return {name: torch.stack(v) if name in ("grad_wg", "grad_wu") else torch.cat(v) for name, v in found.items()}
