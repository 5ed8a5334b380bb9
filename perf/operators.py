"""Performance cases of the expert operators: routing, ragged products grouped by
expert with their gradients, the weighted sum back to tokens, and products in
8-bit integers.

Each case is one call (or the short sequence of calls) that a program makes
through the public entry points of einjax_amd on data resident on the GPU.
``own`` selects the library's operators; where it is false the same results
come from plain torch operations in 32 bits, rounded once at the end.

``listed`` names the cases, ``draw`` gives more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is the call,
``work`` the bytes and operations it cannot do without, ``exact`` the same
outputs from the definitions in 64 bits.

Names: ``t`` tokens, ``k`` experts for each token, ``e`` experts, ``n_in`` and
``n_out`` the extents of a product, a slot is one (token, expert) pair, and
``drop`` the share of tokens without any expert (padding).
"""

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}

# ---------------------------------------------------------------------------
# The cases.


def listed():
    return [
        # Routing of a single token while answering: latency alone.
        dict(name="route_1_e64_k4", kind="route", t=1, e=64, k=4, dtype="fp32", renorm=True,
             grad=False),
        # Routing of a training batch and its gradient.
        dict(name="route_16k_e128_k8_train", kind="route", t=16384, e=128, k=8, dtype="fp32",
             renorm=True, grad=True),
        # Products of a few tokens being answered: the experts' weights are
        # read once and bound the time.  Weights as a linear layer keeps them
        # (one row for each output channel).
        dict(name="grouped_16_e16_bf16", kind="grouped", t=16, e=16, k=2, n_in=2048, n_out=4096,
             order="nk", gather=True, skew=0.3, drop=0.0, dtype="bf16"),
        # A prompt of odd length through experts of odd extents, unevenly
        # chosen: no row starts on a 16-byte boundary.
        dict(name="grouped_1511_e12_odd_fp16", kind="grouped", t=1511, e=12, k=2, n_in=771,
             n_out=1283, order="kn", gather=True, skew=0.8, drop=0.0, dtype="fp16"),
        # The largest product: a batch of prompts, four experts for each token.
        dict(name="grouped_8k_k4_e16_bf16", kind="grouped", t=8192, e=16, k=4, n_in=4096,
             n_out=4096, order="kn", gather=True, skew=0.3, drop=0.0, dtype="bf16"),
        # Rows already grouped, in fp32.
        dict(name="grouped_2k_e8_fp32", kind="grouped", t=2048, e=8, k=2, n_in=1024, n_out=2048,
             order="kn", gather=False, skew=0.3, drop=0.0, dtype="fp32"),
        # A training step of the product: forward and both gradients.
        dict(name="train_8k_e16_bf16", kind="train", t=8192, e=16, k=2, n_in=2048, n_out=4096,
             order="kn", gather=True, skew=0.3, drop=0.0, dtype="bf16"),
        # The same on a small fp32 layer with uneven experts and padded tokens.
        dict(name="train_600_e5_fp32", kind="train", t=600, e=5, k=2, n_in=320, n_out=520,
             order="nk", gather=True, skew=1.0, drop=0.1, dtype="fp32"),
        # The weighted sum of a few tokens' expert results.
        dict(name="combine_8_k4_bf16", kind="combine", t=8, e=16, k=4, n_out=2048, skew=0.3,
             drop=0.0, dtype="bf16", grad=False),
        # The same for a training batch, with the gradients of values and weights.
        dict(name="combine_16k_k4_bf16_train", kind="combine", t=16384, e=64, k=4, n_out=4096,
             skew=0.3, drop=0.05, dtype="bf16", grad=True),
        # 8-bit weights of one dense layer applied to a few tokens.
        dict(name="int8_4_dense_bf16", kind="int8", t=4, e=1, k=1, n_in=4096, n_out=8192,
             gather=False, skew=0.0, drop=0.0, dtype="bf16"),
        # 8-bit experts on a batch of prompts.
        dict(name="int8_8k_k2_e8_bf16", kind="int8", t=8192, e=8, k=2, n_in=4096, n_out=4096,
             gather=True, skew=0.3, drop=0.0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _extent(rng, lo, hi):
    """Half the extents are multiples of 64, a quarter of 8, the rest anything."""
    v = _log_int(rng, lo, hi)
    r = rng.random()
    return max(lo, v // 64 * 64) if r < 0.5 else max(lo, v // 8 * 8) if r < 0.75 else v


def _draw_once(rng):
    kind = rng.choice(("route", "route", "grouped", "grouped", "grouped", "train", "train",
                       "combine", "int8", "int8"))
    if kind == "route":
        e = _log_int(rng, 4, 128)
        return dict(kind=kind, t=_log_int(rng, 1, 16384), e=e, k=rng.randint(1, min(8, e)),
                    dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")),
                    renorm=rng.random() < 0.7, grad=rng.random() < 0.5)
    if kind == "combine":
        e = _log_int(rng, 4, 128)
        return dict(kind=kind, t=_log_int(rng, 1, 16384), e=e, k=rng.randint(1, 4),
                    n_out=_extent(rng, 64, 4096), skew=rng.choice((0.0, 0.3, 0.8)),
                    drop=rng.choice((0.0, 0.0, 0.05, 0.2)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), grad=rng.random() < 0.5)
    e = _log_int(rng, 1, 64)
    c = dict(kind=kind, t=_log_int(rng, 1, 8192), e=e, k=rng.randint(1, min(4, e)),
             n_in=_extent(rng, 64, 4096), n_out=_extent(rng, 64, 4096),
             gather=rng.random() < 0.6, skew=rng.choice((0.0, 0.3, 0.8)),
             drop=rng.choice((0.0, 0.0, 0.1)))
    if kind == "int8":
        return dict(c, dtype=rng.choice(("bf16", "fp16", "fp32")))
    return dict(c, order=rng.choice(("kn", "nk")),
                dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        for key in m:
            m[key] = max(m[key], w[key])
    while True:
        c = _draw_once(rng)
        w, m = work(c), most[c["kind"]]
        # fp32 products run at a fraction of the 16-bit rate
        scale = 8 if c["dtype"] == "fp32" and c["kind"] in ("grouped", "train") else 1
        if w["bytes"] <= m["bytes"] and w["flops"] * scale <= m["flops"]:
            return c


def work(case):
    t, e, k = case["t"], case["e"], case["k"]
    s, b = t * k, _BYTES[case["dtype"]]
    if case["kind"] == "route":
        # logits in; weights, experts, rows and slots out; with the gradient
        # the logits, experts and the weights' gradient in, the logits' out
        bytes_ = t * e * b + 16 * s + 4 * (e + 1)
        flops = 3 * t * e
        if case["grad"]:
            bytes_ += 2 * t * e * b + 8 * s
            flops += 4 * t * e
        return {"bytes": bytes_, "flops": flops}
    live = t - int(t * case["drop"])
    n = case["n_out"]
    sl = live * k
    if case["kind"] == "combine":
        bytes_ = sl * n * b + 8 * s + t * n * b
        flops = 2 * sl * n
        if case["grad"]:
            bytes_ += t * n * b + sl * n * b + 8 * s + s * n * b + 4 * s
            flops += 3 * sl * n
        return {"bytes": bytes_, "flops": flops}
    ki = case["n_in"]
    rows = t if case["gather"] else s
    experts = min(e, sl)
    if case["kind"] == "int8":
        # activations in their own type, 8-bit weights, scales, results
        return {"bytes": rows * ki * b + experts * n * (ki + 4) + s * n * b,
                "flops": 2 * sl * ki * n}
    x, w, y = rows * ki * b, experts * ki * n * b, s * n * b
    if case["kind"] == "grouped":
        return {"bytes": x + w + y, "flops": 2 * sl * ki * n}
    # forward; the gradient of x; the gradient of every expert's weights
    return {"bytes": (x + w + y) + (y + w + x) + (x + y + e * ki * n * b),
            "flops": 6 * sl * ki * n}


# ---------------------------------------------------------------------------
# What a program holds before the call.


def _picks(case, g):
    """Experts [t, k] of each token: distinct, some chosen more often than
    others, -1 for tokens that are padding."""
    t, e, k = case["t"], case["e"], case["k"]
    popular = case["skew"] * torch.randn(e, generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
    experts = torch.sort(popular + noise, dim=1, descending=True).indices[:, :k]
    dropped = int(t * case["drop"])
    if dropped:
        experts[torch.randperm(t, generator=g, device="cuda")[:dropped]] = -1
    return experts


def _group(experts, e):
    """offsets [e + 1], rows [t * k] and slots [t, k] of the pairs sorted by
    expert, pairs of one expert in the order of their tokens; pairs without an
    expert have slot -1 and no row (0)."""
    t, k = experts.shape
    flat = experts.reshape(-1)
    key = torch.where(flat < 0, torch.full_like(flat, e), flat)
    order = torch.sort(key, stable=True).indices
    ends = torch.cumsum(torch.bincount(key, minlength=e + 1)[:e], 0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k, device=flat.device)
    slots = torch.where(flat < 0, torch.full_like(place, -1), place).reshape(t, k)
    rows = torch.where(torch.arange(t * k, device=flat.device) < offsets[e],
                       torch.div(order, k, rounding_mode="floor"), torch.zeros_like(order))
    return offsets.int(), rows.int(), slots.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, e, k, dt = case["t"], case["e"], case["k"], _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    s = dict(case=case)
    if case["kind"] == "route":
        s["logits"] = normal(t, e, scale=1.5).to(dt)
        s["grad"] = normal(t, k)
        return s
    experts = _picks(case, g)
    offsets, rows, slots = _group(experts, e)
    weights = torch.rand(t, k, generator=g, device="cuda")
    weights = torch.where(experts < 0, torch.zeros_like(weights),
                          weights / weights.sum(1, keepdim=True))
    # rows and slots that belong to no expert: row 0, slot -1
    s.update(experts=experts.int(), offsets=offsets, rows=rows, slots=slots, weights=weights)
    n = case["n_out"]
    if case["kind"] == "combine":
        s["y"] = normal(t * k, n).to(dt)
        s["grad"] = normal(t, n).to(dt)
        return s
    ki = case["n_in"]
    s["x"] = normal(t if case["gather"] else t * k, ki).to(dt)
    # The slots of every expert as one rectangle, for products of equal size:
    # the slot at each place (0 where an expert has fewer), whether there is
    # one, and the place of each slot.
    sizes = (offsets[1:] - offsets[:-1]).long()
    most = max(1, int(sizes.max()))
    at = torch.arange(most, device="cuda")
    s["held"] = at < sizes[:, None]
    s["box"] = torch.where(s["held"], offsets[:-1, None].long() + at, 0)
    slot = torch.arange(t * k, device="cuda")
    owner = torch.searchsorted(offsets[1:].long(), slot, right=True).clamp(max=e - 1)
    s["place"] = owner * most + (slot - offsets[owner].long()).clamp(max=most - 1)
    s["live"] = slot < offsets[e]
    w = normal(e, ki, n, scale=ki ** -0.5)
    if case["kind"] == "int8":
        scale = w.abs().amax(1) * (1.0 / 127.0)
        s["w"] = torch.round(w / scale[:, None, :]).clamp(-127, 127).to(torch.int8) \
            .transpose(1, 2).contiguous()
        s["w_scale"] = scale
        return s
    w = w.to(dt)
    s["w"] = w if case["order"] == "kn" else w.transpose(1, 2).contiguous().transpose(1, 2)
    if case["kind"] == "train":
        s["grad"] = normal(t * k, n).to(dt)
    return s


# ---------------------------------------------------------------------------
# The call.


def run(state):
    kind = state["case"]["kind"]
    return (_run_own if own else _run_plain)[kind](state)


def _routing(ej, s):
    return ej.ExpertRouting(weights=s["weights"], experts=s["experts"], offsets=s["offsets"],
                            rows=s["rows"], slots=s["slots"])


def _own_route(s):
    import einjax_amd as ej

    c = s["case"]
    logits = s["logits"].detach().requires_grad_(c["grad"])
    r = ej.route_experts(logits, c["k"], renormalize=c["renorm"])
    out = [r.weights.detach(), r.experts, r.offsets, r.rows, r.slots]
    if c["grad"]:
        out.append(torch.autograd.grad(r.weights, logits, s["grad"])[0])
    return out


def _own_grouped(s):
    import einjax_amd as ej

    return ej.grouped_matmul(s["x"], s["w"], _routing(ej, s), gather=s["case"]["gather"])


def _own_train(s):
    import einjax_amd as ej

    x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
    y = ej.grouped_matmul(x, w, _routing(ej, s), gather=s["case"]["gather"])
    return [y.detach(), *torch.autograd.grad(y, (x, w), s["grad"])]


def _own_combine(s):
    import einjax_amd as ej

    if not s["case"]["grad"]:
        return ej.combine_experts(s["y"], _routing(ej, s))
    y, weights = s["y"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    out = ej.combine_experts(y, _routing(ej, s), weights)
    return [out.detach(), *torch.autograd.grad(out, (y, weights), s["grad"])]


def _own_int8(s):
    import einjax_amd as ej

    c = s["case"]
    q, scale = ej.quantize_rows(s["x"])
    # a single matrix without padded tokens is the dense product
    groups = None if c["e"] == 1 and not c["drop"] else _routing(ej, s)
    return ej.int8_matmul(q, scale, s["w"], s["w_scale"], groups, out_dtype=_DTYPES[c["dtype"]],
                          gather=c["gather"] and groups is not None)


# The plain forms.


def _plain_route(s):
    c = s["case"]
    k, e = c["k"], c["e"]
    l32 = s["logits"].float()
    p = torch.exp(l32 - l32.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    experts = torch.sort(l32, dim=1, descending=True, stable=True).indices[:, :k]
    picked = p.gather(1, experts)
    weights = picked / picked.sum(1, keepdim=True) if c["renorm"] else picked
    out = [weights, experts.int(), *_group(experts, e)]
    if c["grad"]:
        g = s["grad"]
        dot = (weights * g).sum(1, keepdim=True)
        if c["renorm"]:
            d = torch.zeros_like(l32).scatter(1, experts, weights * (g - dot))
        else:
            d = p * (torch.zeros_like(l32).scatter(1, experts, g) - dot)
        out.append(d.to(s["logits"].dtype))
    return out


def _boxes(s, v, gather):
    """v's rows as [e, most, extent] in 32 bits, zero where an expert has fewer."""
    at = s["rows"].long()[s["box"]] if gather else s["box"]
    return v[at].float() * s["held"][..., None]


def _slots_of(s, boxes):
    """[e, most, extent] back to the slots in order, zero past the last live one."""
    return boxes.reshape(-1, boxes.shape[-1])[s["place"]] * s["live"][:, None]


def _to_tokens(s, v):
    """The sum of each token's live slots."""
    slots = s["slots"].long()
    return (v[slots.clamp(min=0)] * (slots >= 0)[..., None]).sum(1)


def _plain_grouped(s):
    y = _slots_of(s, torch.bmm(_boxes(s, s["x"], s["case"]["gather"]), s["w"].float()))
    return y.to(s["x"].dtype)


def _plain_train(s):
    gather, dt = s["case"]["gather"], s["x"].dtype
    x, w, g = _boxes(s, s["x"], gather), s["w"].float(), _boxes(s, s["grad"], False)
    y = _slots_of(s, torch.bmm(x, w))
    dx = _slots_of(s, torch.bmm(g, w.transpose(1, 2)))
    dw = torch.bmm(x.transpose(1, 2), g)
    return [y.to(dt), (_to_tokens(s, dx) if gather else dx).to(dt), dw.to(dt)]


def _plain_combine(s):
    slots, w = s["slots"].long(), s["weights"]
    held = (slots >= 0)[..., None]
    y = s["y"][slots.clamp(min=0)].float() * held
    out = (w[..., None] * y).sum(1).to(s["y"].dtype)
    if not s["case"]["grad"]:
        return out
    g = s["grad"].float()
    # pairs without a slot write a row past the last one
    n = len(s["y"])
    dy = torch.zeros(n + 1, g.shape[1], device=g.device)
    dy[torch.where(slots < 0, n, slots).reshape(-1)] = \
        (w[..., None] * g[:, None, :]).reshape(-1, g.shape[1])
    dy = dy[:n]
    return [out, dy.to(s["y"].dtype), (y * g[:, None, :]).sum(2)]


def _plain_int8(s):
    c = s["case"]
    x = s["x"].float()
    scale = x.abs().amax(1) * (1.0 / 127.0)
    q = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), torch.zeros_like(x))
    acc = torch.bmm(_boxes(s, q, c["gather"]), s["w"].float().transpose(1, 2))
    rows = (s["rows"].long() if c["gather"] else torch.arange(len(s["rows"]), device=x.device))
    acc = acc * s["w_scale"][:, None, :]
    return (_slots_of(s, acc) * scale[rows][:, None]).to(_DTYPES[c["dtype"]])


_run_own = dict(route=_own_route, grouped=_own_grouped, train=_own_train, combine=_own_combine,
                int8=_own_int8)
_run_plain = dict(route=_plain_route, grouped=_plain_grouped, train=_plain_train,
                  combine=_plain_combine, int8=_plain_int8)


# ---------------------------------------------------------------------------
# The definitions in 64 bits.


def exact(case, seed):
    s = prepare(case, seed)
    kind, e, k, t = case["kind"], case["e"], case["k"], case["t"]
    if kind == "route":
        logits = s["logits"].double()
        experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
        p = torch.softmax(logits, 1)
        w = p.gather(1, experts)
        if case["renorm"]:
            w = torch.softmax(logits.gather(1, experts), 1)
        out = [w, experts.int(), *_group(experts, e)]
        if case["grad"]:
            g = s["grad"].double()
            # the Jacobian of a softmax applied to g
            if case["renorm"]:
                d = torch.zeros_like(logits)
                d.scatter_(1, experts, w * g - w * (w * g).sum(1, keepdim=True))
            else:
                full = torch.zeros_like(logits).scatter_(1, experts, g)
                d = p * full - p * (p * full).sum(1, keepdim=True)
            out.append(d)
        return out
    ends = s["offsets"].tolist()
    if kind == "combine":
        y, w = s["y"].double(), s["weights"].double()
        n = y.shape[1]
        out = torch.zeros(t, n, dtype=torch.double, device="cuda")
        dy, dw = torch.zeros_like(y), torch.zeros_like(w)
        g = s["grad"].double()
        for j in range(k):
            tok = torch.nonzero(s["slots"][:, j] >= 0)[:, 0]
            at = s["slots"][tok, j].long()
            out[tok] += w[tok, j, None] * y[at]
            dy[at] = w[tok, j, None] * g[tok]
            dw[tok, j] = (y[at] * g[tok]).sum(1)
        return [out, dy, dw] if case["grad"] else out
    x, n = s["x"], case["n_out"]
    rows = s["rows"].long() if case["gather"] else torch.arange(t * k, device="cuda")
    y = torch.zeros(t * k, n, dtype=torch.double, device="cuda")
    if kind == "int8":
        x = x.double()
        scale = x.abs().amax(1) / 127
        q = torch.round(x / torch.where(scale > 0, scale, 1)[:, None])
        for i in range(e):
            at = rows[ends[i]:ends[i + 1]]
            y[ends[i]:ends[i + 1]] = (q[at] @ s["w"][i].double().T) * scale[at, None] \
                * s["w_scale"][i].double()
        return y
    grad = s["grad"] if kind == "train" else None
    dx = torch.zeros(x.shape, dtype=torch.double, device="cuda")
    dw = torch.zeros(s["w"].shape, dtype=torch.double, device="cuda")
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        xi, wi = x[rows[a:b]].double(), s["w"][i].double()
        y[a:b] = xi @ wi
        if grad is not None:
            gi = grad[a:b].double()
            dx.index_add_(0, rows[a:b], gi @ wi.T)
            dw[i] = xi.T @ gi
    return [y, dx, dw] if grad is not None else y
