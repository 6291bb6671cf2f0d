"""Cases for the operators of the dense layers behind the feature transformer.

Three operators of ``stockfish_trainer_b200.layer_stacks`` are covered, each in
its plain form (elementary torch operations in 32 bits, rounded once at the
end) and as a user calls it (``own``):

* ``linear``: out = act(x W^T + b) + residual, and its gradients;
* ``norm``: y = scale * x + gate * norm(f), h = norm(y), and their gradients;
* ``route``: softmax, top-k choice, per-stack counts and balance loss, and the
  gradient of the logits.

Widths are those of the feature transformer (L1 = 1040, 1024) and of the layer
stacks behind it (8 stacks of 16 or 32), batches those of training (16384,
65536) and of evaluating single positions; the rest are generic odd sizes.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _linear(name, rows, inputs, outputs, dtype, act, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "act": act, "residual": residual, "train": train}


def _norm(name, rows, width, dtype, kind, gate, learned_scale, bias, train):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "kind": kind, "gate": gate,
            "learned_scale": learned_scale, "bias": bias, "train": train}


def _route(name, rows, experts, k, dtype, masked, renormalize, train):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "k": k, "dtype": dtype, "masked": masked,
            "renormalize": renormalize, "train": train}


def listed():
    return [
        # one position through the first layer of 8 stacks of 32, as an analysis tool asks for it: latency
        _linear("linear_one_position_fp32", 1, 1040, 256, "fp32", "crelu", False, False),
        # a handful of positions (a search's leaf batch) through a square block in 16 bits
        _linear("linear_leaf_batch_bf16", 24, 1040, 1040, "bf16", "silu", True, False),
        # validation: forward only over the default training batch, 8 stacks of 16
        _linear("linear_validate_fp32", 16384, 1040, 128, "fp32", "sqr_crelu", False, False),
        # training step of the first layer at the recipe's batch, all stacks' outputs at once
        _linear("linear_train_first_layer_fp32", 65536, 1040, 256, "fp32", "silu", False, True),
        # training step of a residual block's square layer at the recipe's batch: the largest
        _linear("linear_train_block_bf16", 65536, 1040, 1040, "bf16", "gelu", True, True),
        # odd sizes: rows that start at no 16-byte boundary, ragged tiles on every side
        _linear("linear_train_odd_fp16", 4099, 517, 331, "fp16", "gelu", True, True),
        # one position through the norms around a block: latency
        _norm("norm_one_position_bf16", 1, 1040, "bf16", "rms", "row", False, False, False),
        # training step of the norms around a routed block at the recipe's batch
        _norm("norm_train_routed_block_fp32", 65536, 1040, "fp32", "rms", "row", False, False, True),
        # layer norm with biases, an elementwise sigmoid gate, a learned scale, an odd width
        _norm("norm_train_gated_odd_bf16", 5003, 1031, "bf16", "layer", "full", True, True, True),
        # the router over 8 stacks at the recipe's batch, with the balance loss's gradient
        _route("route_train_8_stacks_fp32", 65536, 8, 2, "fp32", False, True, True),
        # many experts, some closed to a position, positions left out of the batch, odd count
        _route("route_train_many_masked_bf16", 9001, 67, 3, "bf16", True, False, True),
        # a few positions being routed, forward only: latency
        _route("route_leaf_batch_fp32", 24, 8, 1, "fp32", False, False, False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: two in three a multiple of 8, as a network's are, the rest any."""
    n = _log_int(rng, lo, hi)
    if n >= 8 and rng.random() < 2 / 3:
        n = min(hi, (n + 7) // 8 * 8)
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "route"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.7
    if op == "linear":
        inputs, outputs = _width(rng, 16, 2080), _width(rng, 1, 1040)
        # fp32 work counts six times: the listed fp32 step is the bound there
        cap = 65536 * 1040 * (256 if dtype == "fp32" else 1040) // (inputs * outputs)
        rows = _log_int(rng, 1, max(1, min(65536, cap)))
        acts = ["none", "silu", "gelu"] if train else ["none", "silu", "gelu", "relu", "crelu", "sqr_crelu"]
        case = _linear("", rows, inputs, outputs, dtype, rng.choice(acts), rng.random() < 0.5, train)
    elif op == "norm":
        width = _width(rng, 16, 4096)
        rows = _log_int(rng, 1, min(65536, 65536 * 1040 // width))
        case = _norm("", rows, width, dtype, rng.choice(["rms", "layer"]), rng.choice(["none", "row", "full"]),
                     rng.random() < 0.5, rng.random() < 0.5, train)
    else:
        experts = _log_int(rng, 2, 256)
        rows = _log_int(rng, 1, 65536 * 64 // max(experts, 64))
        case = _route("", rows, experts, rng.randint(1, min(8, experts)), dtype, rng.random() < 0.5,
                      rng.random() < 0.5, train)
    del case["name"]
    for key in ("rows", "inputs", "outputs", "width"):
        if case.get(key) == 3072:
            case[key] = 3071
    return case


# ---- inputs ----------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _inputs(case, seed):
    """The inputs of a case as plain tensors (no gradients asked for)."""
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]
    B = case["rows"]
    s = {}
    if case["op"] == "linear":
        K, N = case["inputs"], case["outputs"]
        if case["act"] in ("crelu", "sqr_crelu"):
            # what the feature transformer's epilogue hands over: products of two values clamped to [0, 1]
            a = (_randn(g, B, K) * 0.5 + 0.3).clamp_(0, 1)
            s["x"] = (a * (_randn(g, B, K) * 0.5 + 0.3).clamp_(0, 1) * (127 / 128)).to(dt)
        else:
            s["x"] = _randn(g, B, K).to(dt)
        s["weight"] = ((torch.rand(N, K, generator=g, device="cuda") * 2 - 1) * math.sqrt(3.0 / K)).to(dt)
        s["bias"] = (_randn(g, N) * 0.1).to(dt)
        s["residual"] = _randn(g, B, N).to(dt) if case["residual"] else None
        if case["train"]:
            s["grad_out"] = _randn(g, B, N).to(dt)
    elif case["op"] == "norm":
        D = case["width"]
        s["x"] = _randn(g, B, D).to(dt)
        s["f"] = (_randn(g, B, D) * 3.0 + 0.1).to(dt)
        s["post_weight"] = 1 + 0.1 * _randn(g, D)
        s["pre_weight"] = 1 + 0.1 * _randn(g, D)
        s["post_bias"] = 0.1 * _randn(g, D) if case["bias"] else None
        s["pre_bias"] = 0.1 * _randn(g, D) if case["bias"] else None
        s["scale"] = 0.9 + 0.1 * _randn(g, D) if case["learned_scale"] else None
        s["gate"] = None
        if case["gate"] == "row":  # a router's gate per position
            s["gate"] = torch.rand(B, generator=g, device="cuda") * 0.9 + 0.1
        elif case["gate"] == "full":  # the branch's own gate values, through a sigmoid
            s["gate"] = _randn(g, B, D).to(dt)
        if case["train"]:
            s["grad_y"] = _randn(g, B, D).to(dt)
            s["grad_h"] = _randn(g, B, D).to(dt)
    else:
        E, k = case["experts"], case["k"]
        logits = _randn(g, B, E) * 1.5 + 0.5 * _randn(g, E)
        s["valid"] = None
        if case["masked"]:
            # stacks closed to a position, one row in 16 with none open, one in 8 left out of the batch
            closed = torch.rand(B, E, generator=g, device="cuda") < 0.25
            closed |= torch.rand(B, 1, generator=g, device="cuda") < 1 / 16
            logits = logits.masked_fill(closed, float("-inf"))
            s["valid"] = torch.rand(B, generator=g, device="cuda") >= 1 / 8
        s["logits"] = logits.to(dt)
        if case["train"]:
            s["grad_gates"] = _randn(g, B, k)
            s["grad_loss"] = torch.full((), 0.01 * B, device="cuda")
    return s


_LEAVES = {"linear": ("x", "weight", "bias", "residual"),
           "norm": ("x", "f", "post_weight", "post_bias", "gate", "scale", "pre_weight", "pre_bias"),
           "route": ("logits",)}


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["train"]:
        for name in _LEAVES[case["op"]]:
            if state[name] is not None:
                state[name].requires_grad_()
    state["case"] = case
    return state


# ---- the framework's operators ---------------------------------------------
def _run_own(s):
    from stockfish_trainer_b200 import layer_stacks

    case = s["case"]
    if case["op"] == "linear":
        outs = [layer_stacks.linear_act(s["x"], s["weight"], s["bias"], residual=s["residual"],
                                        activation=case["act"])]
        grads = [s.get("grad_out")]
    elif case["op"] == "norm":
        outs = list(layer_stacks.block_norm(
            s["x"], s["f"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
            gate_activation="sigmoid" if case["gate"] == "full" else "none",
            residual_scale=1.0 if s["scale"] is None else s["scale"], pre_weight=s["pre_weight"],
            pre_bias=s["pre_bias"], kind=case["kind"], eps=1e-5))
        grads = [s.get("grad_y"), s.get("grad_h")]
    else:
        r = layer_stacks.route(s["logits"], case["k"], valid=s["valid"], renormalize=case["renormalize"])
        if not case["train"]:
            return [r.indices, r.gates, r.counts, r.balance_loss]
        d = torch.autograd.grad([r.gates, r.balance_loss], [s["logits"]], [s["grad_gates"], s["grad_loss"]])
        return [r.indices, r.gates.detach(), r.counts, r.balance_loss.detach(), *d]
    if not case["train"]:
        return outs
    leaves = [s[name] for name in _LEAVES[case["op"]] if s[name] is not None]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads))


# ---- the plain forms -------------------------------------------------------
def _act_plain(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).float()
    if act == "crelu":
        return torch.clamp(z, 0, 1), ((z > 0) & (z < 1)).float()
    if act == "sqr_crelu":
        c = torch.clamp(z, 0, 1)
        return c * c, torch.where((z > 0) & (z < 1), 2 * z, 0.0)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return z * sg, sg * (1 + z * (1 - sg))
    phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _plain_linear(s):
    case = s["case"]
    dt = _DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t() + s["bias"].float()
    out, d = _act_plain(z, case["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    outs = [out.to(dt)]
    if case["train"]:
        g = s["grad_out"].float()
        dz = g * d
        outs += [(dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt)]
        if s["residual"] is not None:
            outs.append(s["grad_out"].clone())
    return outs


def _normalise(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((v * v).mean(1, keepdim=True) + eps)
    return v * r, r


def _normalise_back(dv, hat, r, kind):
    """Gradient of the normalised rows' input: ``dv`` belongs to ``hat``."""
    out = dv - hat * (dv * hat).mean(1, keepdim=True)
    if kind == "layer":
        out = out - dv.mean(1, keepdim=True)
    return out * r


def _plain_norm(s):
    case, kind, eps = s["case"], s["case"]["kind"], 1e-5
    dt = _DTYPES[case["dtype"]]
    x, f = s["x"].float(), s["f"].float()
    wp, wn = s["post_weight"], s["pre_weight"]
    scale = 1.0 if s["scale"] is None else s["scale"]
    gate = 1.0
    if case["gate"] == "row":
        gate = s["gate"][:, None]
    elif case["gate"] == "full":
        gate = 1 / (1 + torch.exp(-s["gate"].float()))
    fh, rf = _normalise(f, kind, eps)
    n = fh * wp
    if s["post_bias"] is not None:
        n = n + s["post_bias"]
    y = scale * x + gate * n
    yh, ry = _normalise(y, kind, eps)
    h = yh * wn
    if s["pre_bias"] is not None:
        h = h + s["pre_bias"]
    outs = [y.to(dt), h.to(dt)]
    if not case["train"]:
        return outs
    dh = s["grad_h"].float()
    dy = s["grad_y"].float() + _normalise_back(dh * wn, yh, ry, kind)
    dn = gate * dy
    outs += [(scale * dy).to(dt), _normalise_back(dn * wp, fh, rf, kind).to(dt), (dn * fh).sum(0)]
    if s["post_bias"] is not None:
        outs.append(dn.sum(0))
    if case["gate"] == "row":
        outs.append((dy * n).sum(1))
    elif case["gate"] == "full":
        outs.append((dy * n * gate * (1 - gate)).to(dt))
    if s["scale"] is not None:
        outs.append((dy * x).sum(0))
    outs.append((dh * yh).sum(0))
    if s["pre_bias"] is not None:
        outs.append(dh.sum(0))
    return outs


def _plain_route(s):
    case = s["case"]
    k, E = case["k"], case["experts"]
    raw = s["logits"]
    l = raw.float()
    rows = (l > float("-inf")).any(1)
    if s["valid"] is not None:
        rows = rows & s["valid"]
    m = torch.where(rows[:, None], l, 0.0).max(1, keepdim=True).values
    e = torch.where(rows[:, None], torch.exp(l - m), 0.0)
    p = e / torch.where(rows, e.sum(1), 1.0)[:, None]
    val, idx = torch.sort(l, dim=1, descending=True, stable=True)
    val, idx = val[:, :k], idx[:, :k]
    taken = rows[:, None] & (val > float("-inf"))
    gates = torch.where(taken, torch.gather(p, 1, idx), 0.0)
    total = gates.sum(1, keepdim=True)
    if case["renormalize"]:
        gates = gates / torch.where(total > 0, total, 1.0)
    indices = torch.where(taken, idx, -1)
    counts = (indices[:, :, None] == torch.arange(E, device=l.device)).sum((0, 1)) if E * k * len(l) < 1 << 24 else \
        torch.stack([(indices == i).sum() for i in range(E)])
    n = rows.sum().float().clamp(min=1)
    c = counts.float()
    unit = E / (k * n * n)
    loss = unit * (c * p.sum(0)).sum()
    outs = [indices, gates, counts, loss]
    if case["train"]:
        dg = torch.where(taken, s["grad_gates"], 0.0)
        inner = (dg * gates).sum(1, keepdim=True)
        dl = unit * s["grad_loss"] * p * (c - (p * c).sum(1, keepdim=True))
        if case["renormalize"]:
            dl = dl.scatter_add(1, idx, torch.where(taken, gates * (dg - inner), 0.0))
        else:
            dl = dl - p * inner
            dl = dl.scatter_add(1, idx, gates * dg)
        outs.append(dl.to(raw.dtype))
    return outs


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "route": _plain_route}[state["case"]["op"]](state)


# ---- the definition in 64 bits, by automatic differentiation -----------------
def _act_exact(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    if act == "crelu":
        return z.clamp(0, 1)
    if act == "sqr_crelu":
        return z.clamp(0, 1).square()
    if act == "silu":
        return z * torch.sigmoid(z)
    return z * torch.special.ndtr(z)


def _norm_exact(v, kind, eps):
    if kind == "layer":
        c = v - v.mean(dim=1, keepdim=True)
        return c / torch.sqrt(c.pow(2).mean(dim=1, keepdim=True) + eps)
    return v / torch.sqrt(v.pow(2).mean(dim=1, keepdim=True) + eps)


def exact(case, seed):
    s = {name: t.double() if t is not None and t.is_floating_point() else t
         for name, t in _inputs(case, seed).items()}
    if case["train"]:
        for name in _LEAVES[case["op"]]:
            if s[name] is not None:
                s[name].requires_grad_()
    leaves = [s[name] for name in _LEAVES[case["op"]] if s[name] is not None]
    if case["op"] == "linear":
        out = _act_exact(torch.addmm(s["bias"], s["x"], s["weight"].t()), case["act"])
        if s["residual"] is not None:
            out = out + s["residual"]
        outs, grads = [out], [s.get("grad_out")]
    elif case["op"] == "norm":
        n = _norm_exact(s["f"], case["kind"], 1e-5) * s["post_weight"]
        if s["post_bias"] is not None:
            n = n + s["post_bias"]
        if case["gate"] == "row":
            n = n * s["gate"].unsqueeze(1)
        elif case["gate"] == "full":
            n = n * torch.sigmoid(s["gate"])
        y = s["x"] * (1.0 if s["scale"] is None else s["scale"]) + n
        h = _norm_exact(y, case["kind"], 1e-5) * s["pre_weight"]
        if s["pre_bias"] is not None:
            h = h + s["pre_bias"]
        outs, grads = [y, h], [s.get("grad_y"), s.get("grad_h")]
    else:
        k, E, l = case["k"], case["experts"], s["logits"]
        open_ = torch.isfinite(l.detach())
        rows = open_.any(dim=1) if s["valid"] is None else open_.any(dim=1) & s["valid"]
        open_ = open_ & rows.unsqueeze(1)
        # rows that count, as a softmax over their open entries; the others never enter
        at = rows.nonzero().squeeze(1)
        p = torch.zeros_like(l).index_copy(0, at, torch.softmax(l.index_select(0, at), dim=1))
        order = torch.argsort(l.detach(), dim=1, descending=True, stable=True)[:, :k]
        taken = open_.gather(1, order)
        gates = p.gather(1, order) * taken
        if case["renormalize"]:
            gates = gates / gates.sum(dim=1, keepdim=True).masked_fill(~rows.unsqueeze(1), 1.0)
        indices = order.masked_fill(~taken, -1)
        counts = torch.bincount(order[taken], minlength=E)
        n = max(1, int(rows.sum()))
        loss = E * torch.dot(counts.double() / (k * n), p.sum(dim=0) / n)
        outs = [indices, gates.detach(), counts, loss.detach()]
        if case["train"]:
            outs += torch.autograd.grad([gates, loss], leaves, [s["grad_gates"], s["grad_loss"]])
        return outs
    if not case["train"]:
        return outs
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, grads))


# ---- what a pass cannot do without ------------------------------------------
def work(case):
    e, B = _BYTES[case["dtype"]], case["rows"]
    if case["op"] == "linear":
        K, N = case["inputs"], case["outputs"]
        nbytes = e * (B * K + N * K + N + B * N * (2 if case["residual"] else 1))
        flops = 2 * B * N * K + 4 * B * N
        if case["train"]:  # reads the output's gradient; writes those of x, weight and bias
            nbytes += e * (B * N + B * K + N * K + N)
            flops += 4 * B * N * K + 4 * B * N
    elif case["op"] == "norm":
        D = case["width"]
        per_row = D if case["gate"] == "full" else 0
        nbytes = e * B * (4 * D + per_row)
        flops = 12 * B * D
        if case["train"]:  # two gradients in; those of x, f and the gate out
            nbytes += e * B * (4 * D + per_row)
            flops += 24 * B * D
        params = 2 + 2 * case["bias"] + case["learned_scale"]
        nbytes += 4 * params * D * (2 if case["train"] else 1)
        if case["gate"] == "row":
            nbytes += 4 * B * (2 if case["train"] else 1)
    else:
        E, k = case["experts"], case["k"]
        nbytes = B * (E * e + 12 * k + (1 if case["masked"] else 0)) + 8 * E
        flops = 5 * B * E + 2 * B * E * k
        if case["train"]:
            nbytes += B * (E * e + 4 * k)
            flops += 6 * B * E
    return {"bytes": nbytes, "flops": flops}
