"""The FP8 operators' measured cases, their plain forms and their exact values.

Every operator works on e4m3 values with FP32 scales: activations carry one
scale per row and 128 columns, weights one per 128 x 128 block.

  norm     residual addition, root-mean-square norm and e4m3 output with scales
           (or, without the norm, the e4m3 form of given rows)
  blocks   BF16 weights to e4m3 with a scale per 128 x 128 block
  linear   the matrix product of e4m3 rows with an e4m3 weight
  experts  the routed SwiGLU experts on e4m3 banks: rows to their experts, two
           products with the activation between them kept in e4m3, weighted sum
"""

import torch

own = False

B = 128          # values that share a scale
TOP = 448.0      # the largest e4m3 value
TINY = 1e-10     # a group's maximum counts as at least this


def listed():
    return [
        # one token of a decode step, before its MoE block
        {"name": "norm_token", "op": "norm", "tokens": 1, "hidden": 2048, "norm": True, "residual": True},
        # an odd batch of a model whose width ends inside a group
        {"name": "norm_ragged", "op": "norm", "tokens": 333, "hidden": 1000, "norm": True, "residual": False},
        # a long prompt's rows
        {"name": "norm_prefill", "op": "norm", "tokens": 8192, "hidden": 2048, "norm": True, "residual": True},
        # a single matrix with cut blocks at both edges
        {"name": "blocks_ragged", "op": "blocks", "banks": 1, "rows": 1000, "cols": 2000},
        # one layer's gate/up bank when a BF16 model is loaded
        {"name": "blocks_bank", "op": "blocks", "banks": 256, "rows": 1024, "cols": 2048},
        # the gate and up rows of one expert-sized MLP for one token
        {"name": "linear_token", "op": "linear", "tokens": 1, "rows": 1024, "cols": 2048, "f32": False},
        # a ragged batch, an output width that ends inside a block, FP32 out
        {"name": "linear_ragged", "op": "linear", "tokens": 77, "rows": 1000, "cols": 1040, "f32": True},
        # a projection of a long prompt
        {"name": "linear_prefill", "op": "linear", "tokens": 8192, "rows": 4096, "cols": 2048, "f32": False},
        # one decoded token through a layer's experts
        {"name": "experts_token", "op": "experts", "tokens": 1, "experts": 256, "top_k": 8, "hidden": 2048,
         "inner": 512, "dropped": 0.0},
        # a decode batch
        {"name": "experts_batch", "op": "experts", "tokens": 16, "experts": 256, "top_k": 8, "hidden": 2048,
         "inner": 512, "dropped": 0.0},
        # an odd batch on a shard that holds a part of the routed experts: other routes are dropped
        {"name": "experts_shard", "op": "experts", "tokens": 333, "experts": 64, "top_k": 8, "hidden": 2048,
         "inner": 512, "dropped": 0.5},
        # a prompt
        {"name": "experts_prefill", "op": "experts", "tokens": 4096, "experts": 256, "top_k": 8, "hidden": 2048,
         "inner": 512, "dropped": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "blocks", "linear", "experts"])
    if op == "norm":
        hidden = _log(rng, 128, 8192)
        return {"op": op, "tokens": _log(rng, 1, min(16384, 8192 * 2048 // hidden)), "hidden": hidden,
                "norm": rng.random() < 0.75, "residual": rng.random() < 0.5}
    if op == "blocks":
        rows, cols = _log(rng, 64, 4096), _log(rng, 64, 4096)
        return {"op": op, "banks": _log(rng, 1, min(256, 256 * 1024 * 2048 // (rows * cols))), "rows": rows,
                "cols": cols}
    if op == "linear":
        rows, cols = _log(rng, 64, 8192), 16 * _log(rng, 8, 512)
        tokens = _log(rng, 1, max(1, min(16384, 8192 * 4096 * 2048 // (rows * cols))))
        while tokens * (rows + cols) > 8192 * (4096 + 2048):
            tokens = max(1, tokens // 2)
        return {"op": op, "tokens": tokens, "rows": rows, "cols": cols, "f32": rng.random() < 0.25}
    hidden, inner = 16 * _log(rng, 16, 256), 128 * rng.randint(1, 8)
    experts = _log(rng, 8, max(8, min(256, 256 * 512 * 2048 // (hidden * inner))))
    top_k = rng.randint(1, min(8, experts))
    most = 4096 * 8 * 512 * 2048 // (top_k * hidden * inner)
    return {"op": op, "tokens": _log(rng, 1, max(1, min(8192, most, 4096 * 8 * 2048 // (top_k * hidden)))),
            "experts": experts, "top_k": top_k, "hidden": hidden, "inner": inner,
            "dropped": rng.choice([0.0, 0.0, 0.25, 0.75])}


# ------------------------------------------------------------------ inputs ---

def _groups(n):
    return -(-n // B)


def _quantize_rows(x):
    """FP32 rows [..., n] to (e4m3 [..., n], FP32 scales [..., ceil(n / 128)])."""
    n = x.shape[-1]
    wide = torch.nn.functional.pad(x, (0, _groups(n) * B - n)).unflatten(-1, (_groups(n), B))
    top = wide.abs().amax(-1, keepdim=True).clamp(min=TINY)
    q = (wide * TOP / top).clamp(-TOP, TOP).flatten(-2)[..., :n]
    return q.to(torch.float8_e4m3fn), top.squeeze(-1) / TOP


def _quantize_blocks(w):
    """Matrices [b, n, k] to (e4m3 [b, n, k], FP32 scales [b, ceil(n / 128), ceil(k / 128)])."""
    b, n, k = w.shape
    gn, gk = _groups(n), _groups(k)
    wide = torch.nn.functional.pad(w.float(), (0, gk * B - k, 0, gn * B - n)).view(b, gn, B, gk, B)
    top = wide.abs().amax((2, 4), keepdim=True).clamp(min=TINY)
    q = (wide * TOP / top).clamp(-TOP, TOP).view(b, gn * B, gk * B)[:, :n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), (top / TOP).view(b, gn, gk)


def _routes(tokens, experts, top_k, dropped, gen, device):
    """Distinct experts per token, some more popular than others, and their BF16 weights."""
    logits = torch.randn(tokens, experts, generator=gen, device=device)
    logits += 0.5 * torch.randn(experts, generator=gen, device=device)
    v, idx = logits.topk(top_k, dim=-1)
    w = torch.softmax(v, -1).to(torch.bfloat16)
    if dropped:
        idx = torch.where(torch.rand(idx.shape, generator=gen, device=device) < dropped, -1, idx)
    return idx.contiguous(), w.contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    op, bf = case["op"], torch.bfloat16
    s = {"op": op}
    if op == "norm":
        t, h = case["tokens"], case["hidden"]
        # hidden states have a few channels far above the others
        channel = 1 + 15 * (torch.rand(h, generator=gen, device=dev) < 0.01)
        s["x"] = (rand(t, h) * channel).to(bf)
        s["weight"] = (0.3 * rand(h)).to(bf) if case["norm"] else None
        s["residual"] = (2 * rand(t, h) * channel).to(bf) if case["norm"] and case["residual"] else None
        s["out"] = {"q": torch.empty(t, h, dtype=torch.float8_e4m3fn, device=dev),
                    "scale": torch.empty(t, _groups(h), device=dev)}
        if case["norm"]:
            s["out"]["normed"] = torch.empty(t, h, dtype=bf, device=dev)
        if s["residual"] is not None:
            s["out"]["residual"] = torch.empty(t, h, dtype=bf, device=dev)
    elif op == "blocks":
        s["w"] = (0.02 * rand(case["banks"], case["rows"], case["cols"])).to(bf)
    elif op == "linear":
        s["x"], s["xs"] = _quantize_rows(rand(case["tokens"], case["cols"]))
        s["w"], s["ws"] = (v[0] for v in _quantize_blocks(0.02 * rand(1, case["rows"], case["cols"])))
        s["out"] = torch.empty(case["tokens"], case["rows"], dtype=torch.float32 if case["f32"] else bf, device=dev)
    else:
        e, h, i, t = case["experts"], case["hidden"], case["inner"], case["tokens"]
        s["x"], s["xs"] = _quantize_rows(rand(t, h))
        s["gu"], s["gus"] = _quantize_blocks((0.02 * rand(e, 2 * i, h)).to(bf))
        s["dn"], s["dns"] = _quantize_blocks((0.02 * rand(e, h, i)).to(bf))
        s["idx"], s["weights"] = _routes(t, e, case["top_k"], case["dropped"], gen, dev)
        s["out"] = torch.empty(t, h, dtype=bf, device=dev)
    return s


# ------------------------------------------------------------- plain forms ---

def _widen(q, scale):
    """e4m3 rows and their scales as FP32 rows."""
    return q.float() * scale.repeat_interleave(B, -1)[..., :q.shape[-1]]


def _widen_blocks(q, scale):
    return q.float() * scale.repeat_interleave(B, -2)[..., :q.shape[-2], :].repeat_interleave(B, -1)[
        ..., :q.shape[-1]]


def _plain_norm(s):
    if s["weight"] is None:
        q, scale = _quantize_rows(s["x"].float())
        return {"q": q, "scale": scale}
    out = {}
    x = s["x"]
    if s["residual"] is not None:
        x = (x.float() + s["residual"].float()).to(torch.bfloat16)
        out["residual"] = x
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + s["weight"].float())
    out["q"], out["scale"] = _quantize_rows(y)
    out["normed"] = y.to(torch.bfloat16)
    return out


def _plain_experts(s):
    idx, e = s["idx"], s["gu"].shape[0]
    t, k = idx.shape
    inner = s["dn"].shape[2]
    flat = idx.reshape(-1)
    route = torch.nonzero((flat >= 0) & (flat < e)).squeeze(-1)
    out = torch.zeros(t, s["x"].shape[1], device=idx.device)
    if route.numel() == 0:
        return out.to(torch.bfloat16)
    used, group = torch.unique(flat[route], return_inverse=True)
    order = torch.argsort(group, stable=True)
    route, group = route[order], group[order]
    count = torch.bincount(group, minlength=used.numel())
    place = torch.arange(route.numel(), device=idx.device) - (count.cumsum(0) - count)[group]
    rows = torch.zeros(used.numel(), int(count.max()), s["x"].shape[1], device=idx.device)
    rows[group, place] = _widen(s["x"], s["xs"])[route // k]
    gu = torch.bmm(rows, _widen_blocks(s["gu"][used], s["gus"][used]).transpose(1, 2))
    gate, up = gu[..., :inner], gu[..., inner:]
    act = _widen(*_quantize_rows(gate / (1 + torch.exp(-gate)) * up))
    y = torch.bmm(act, _widen_blocks(s["dn"][used], s["dns"][used]).transpose(1, 2))
    out.index_add_(0, route // k, y[group, place] * s["weights"].reshape(-1)[route].float()[:, None])
    return out.to(torch.bfloat16)


def run(state):
    s, op = state, state["op"]
    if own:
        from lightreason_b200 import fp8

        if op == "norm":
            if s["weight"] is None:
                fp8.quantize_rows(s["x"], out=(s["out"]["q"], s["out"]["scale"]))
            else:
                fp8.rmsnorm_quantize(s["x"], s["weight"], s["residual"], eps=1e-6, weight_offset=1.0,
                                     out=(s["out"]["q"], s["out"]["scale"], s["out"]["normed"],
                                          s["out"].get("residual")))
            return s["out"]
        if op == "blocks":
            q, scale = fp8.quantize_blocks(s["w"])
            return {"q": q, "scale": scale}
        if op == "linear":
            return fp8.linear(s["x"], s["xs"], s["w"], s["ws"], out=s["out"])
        return fp8.experts(s["x"], s["xs"], s["gu"], s["gus"], s["dn"], s["dns"], s["idx"], s["weights"],
                           out=s["out"])
    if op == "norm":
        return _plain_norm(s)
    if op == "blocks":
        q, scale = _quantize_blocks(s["w"])
        return {"q": q, "scale": scale}
    if op == "linear":
        return (_widen(s["x"], s["xs"]) @ _widen_blocks(s["w"], s["ws"]).T).to(s["out"].dtype)
    return _plain_experts(s)


# ------------------------------------------------------------------- work ---

def work(case):
    op = case["op"]
    if op == "norm":
        t, h = case["tokens"], case["hidden"]
        per = 2 + 1 + (2 if case["norm"] else 0) + (4 if case["norm"] and case["residual"] else 0)
        return {"bytes": t * h * per + t * _groups(h) * 4 + (2 * h if case["norm"] else 0), "flops": 8 * t * h}
    if op == "blocks":
        b, n, k = case["banks"], case["rows"], case["cols"]
        return {"bytes": b * (3 * n * k + 4 * _groups(n) * _groups(k)), "flops": 3 * b * n * k}
    if op == "linear":
        m, n, k = case["tokens"], case["rows"], case["cols"]
        return {"bytes": m * k + n * k + 4 * _groups(k) * (m + _groups(n)) + m * n * (4 if case["f32"] else 2),
                "flops": 2 * m * n * k}
    e, h, i, t, k = case["experts"], case["hidden"], case["inner"], case["tokens"], case["top_k"]
    # the experts that a batch reaches, from routes of the same distribution
    seen = min(t, 1024)
    idx, _ = _routes(seen, e, k, case["dropped"], torch.Generator().manual_seed(1), "cpu")
    used = int(torch.unique(idx[idx >= 0]).numel()) if seen == t else e
    routes = t * k * (1 - case["dropped"])
    return {"bytes": used * (3 * i * h + 12 * _groups(i) * _groups(h)) + t * (h + 4 * _groups(h) + 2 * h + 10 * k),
            "flops": 6 * routes * i * h}


# ------------------------------------------------------------------ exact ---

def _nearest_e4m3(v):
    """64-bit values to the nearest e4m3 value, ties to the even one: 3 fraction bits down to 2^-6, steps of 2^-9 below."""
    exponent = torch.frexp(v.abs().clamp(min=2.0 ** -6))[1].double() - 1
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_rows(y):
    """64-bit rows: their e4m3 values and scales, group by group."""
    q, scales = [], []
    for c in range(0, y.shape[-1], B):
        part = y[..., c:c + B]
        top = part.abs().amax(-1, keepdim=True).clamp(min=TINY)
        q.append(_nearest_e4m3(part * TOP / top))
        scales.append(top / TOP)
    return torch.cat(q, -1), torch.cat(scales, -1)


def _exact_values(q, scale):
    """What e4m3 values and scales stand for, in 64 bits, column group by column group."""
    return torch.cat([q[..., c:c + B].double() * scale[..., c // B, None].double()
                      for c in range(0, q.shape[-1], B)], -1)


def _exact_matrix(q, scale):
    return torch.cat([_exact_values(q[r:r + B], scale[r // B].expand(min(B, q.shape[0] - r), -1))
                      for r in range(0, q.shape[0], B)], 0)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        x = s["x"].double()
        if s["weight"] is None:
            q, scale = _exact_rows(x)
            return {"q": q, "scale": scale}
        out = {}
        if s["residual"] is not None:
            total = x + s["residual"].double()
            out["residual"] = total
            x = total.to(torch.bfloat16).double()   # the norm is of the sum as it is stored
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * (1 + s["weight"].double())
        out["q"], out["scale"] = _exact_rows(y)
        out["normed"] = y
        return out
    if op == "blocks":
        q, scale = [], []
        for r in range(0, case["rows"], B):
            tops = [s["w"][:, r:r + B, c:c + B].double().abs().amax((1, 2)).clamp(min=TINY)
                    for c in range(0, case["cols"], B)]
            wide = torch.stack(tops, -1)[:, None, :].repeat_interleave(B, -1)[..., :case["cols"]]
            q.append(_nearest_e4m3(s["w"][:, r:r + B].double() * TOP / wide).to(torch.float32))
            scale.append(torch.stack(tops, -1) / TOP)
        return {"q": torch.cat(q, 1), "scale": torch.stack(scale, 1)}
    if op == "linear":
        return _exact_values(s["x"], s["xs"]) @ _exact_matrix(s["w"], s["ws"]).T
    i = case["inner"]
    x = _exact_values(s["x"], s["xs"])
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = torch.nonzero(s["idx"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        gu = x[token] @ _exact_matrix(s["gu"][e], s["gus"][e]).T
        act = gu[:, :i] * torch.sigmoid(gu[:, :i]) * gu[:, i:]
        q, scale = _exact_rows(act)
        y = _exact_values(q, scale) @ _exact_matrix(s["dn"][e], s["dns"][e]).T
        out.index_add_(0, token, y * s["weights"][token, slot].double()[:, None])
    return out
