"""Timing cases of the training operators around the MoE block, their plain forms and their 64-bit results.

Kinds (``case["kind"]``):

* ``aux``    the router's auxiliary loss (balance and z-loss) over all layers' logits, with the
             per-expert counts and every layer's gradient
* ``norm``   layer norm over the last dimension: forward alone, or forward and backward with the
             gradients of weight and bias
* ``save8``  a tensor saved in 8 bits (groups of 32 columns, a power-of-two scale each) and read back
* ``ffn8``   the expert FFN's two products around its 8-bit checkpoint: the gate_up product with its
             SwiGLU, which saves the pre-activations in 8 bits, and in the backward the down product's
             input gradient through the SwiGLU, which reads them and computes the activation again
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# hidden, experts, top-k, expert intermediate of the layers that pluggy_amd.workloads describes
LAYERS = {"climbmix": (1024, 32, 4, 512), "30b-a3b": (2048, 128, 8, 768)}
GROUP = 32  # columns that share a scale


def _aux(layers, tokens, experts, top_k, dtype, masked):
    return {"kind": "aux", "layers": int(layers), "tokens": int(tokens), "experts": int(experts), "top_k": int(top_k),
            "dtype": dtype, "masked": bool(masked)}


def _norm(rows, width, dtype, backward):
    return {"kind": "norm", "rows": int(rows), "width": int(width), "dtype": dtype, "backward": bool(backward)}


def _save8(rows, width, dtype):
    return {"kind": "save8", "rows": int(rows), "width": int(width), "dtype": dtype}


def _ffn8(layer, tokens, dtype):
    return {"kind": "ffn8", "layer": layer, "tokens": int(tokens), "dtype": dtype}


def listed():
    cases = {
        # one layer's loss on a short batch of odd length: launches and host work are most of it
        "aux-1x613": _aux(1, 613, 32, 4, "fp32", False),
        # a padded batch under bf16 logits (equal ones are common there), an expert count that is no power of two
        "aux-6x1531-padded": _aux(6, 1531, 60, 6, "bf16", True),
        # a twelve-layer model's training micro-batch
        "aux-12x8192": _aux(12, 8192, 32, 4, "fp32", False),
        # a deep model of many experts: the largest
        "aux-48x8192": _aux(48, 8192, 128, 8, "fp32", False),
        # a decode batch: latency
        "norm-7x2048": _norm(7, 2048, "bf16", False),
        # an odd width and odd row count in fp32, rows that start at any 4 bytes
        "norm-1531x1001": _norm(1531, 1001, "fp32", True),
        # a training micro-batch
        "norm-8192x2048": _norm(8192, 2048, "bf16", True),
        # a wide layer's long batch
        "norm-16384x4096": _norm(16384, 4096, "bf16", True),
        # a small tensor of odd width
        "save8-520x1001": _save8(520, 1001, "fp32"),
        # the pre-activations of a layer's micro-batch: 65536 pairs of 2 * 768
        "save8-65536x1536": _save8(65536, 1536, "bf16"),
        # a small layer's micro-batch of odd length
        "ffn8-1531": _ffn8("climbmix", 1531, "bf16"),
        # the headline layer's micro-batch: the largest
        "ffn8-8192": _ffn8("30b-a3b", 8192, "bf16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly whole 16-byte rows, one in four of any width."""
    w = _log_uniform(rng, lo, hi)
    return w if rng.random() < 0.25 else (w + 7) // 8 * 8


def draw(rng):
    kind = rng.choice(["aux", "aux", "norm", "norm", "save8", "ffn8"])
    half = "fp16" if rng.random() < 0.3 else "bf16"
    if kind == "aux":
        experts = rng.choice([4, 8, 16, 24, 32, 60, 64, 100, 128, 128, 256])
        layers = _log_uniform(rng, 1, 48)
        tokens = _log_uniform(rng, 1, min(16384, 48 * 8192 * 128 // (layers * experts)))
        return _aux(layers, tokens, experts, rng.randint(1, min(8, experts)), rng.choice(["fp32", "fp32", "bf16"]),
                    rng.random() < 0.3)
    if kind == "norm":
        width = _width(rng, 32, 16384)
        rows = _log_uniform(rng, 1, min(32768, 16384 * 4096 // width))
        return _norm(rows, width, rng.choice(["fp32", half, half]) if rows * width < 16384 * 2048 else half,
                     rng.random() < 0.7)
    if kind == "save8":
        width = _width(rng, 16, 8192)
        rows = _log_uniform(rng, 1, 65536 * 1536 // 2 // width)
        return _save8(rows, width, rng.choice(["fp32", half, half]))
    return _ffn8(rng.choice(list(LAYERS)), _log_uniform(rng, 128, 8191), half)


def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "aux":
        L, N, E = case["layers"], case["tokens"], case["experts"]
        # a trained router: experts of unequal favour, each layer its own
        bias = _randn(gen, L, 1, E, std=0.5)
        logits = [(_randn(gen, N, E) + bias[i]).to(dt).requires_grad_() for i in range(L)]
        mask = None
        if case["masked"]:  # the padded ends of four sequences
            per = -(-N // 4)
            ends = torch.randint(per // 2, per + 1, (4, 1), generator=gen, device=DEV)
            mask = (torch.arange(per, device=DEV) < ends).reshape(-1)[:N].contiguous()
        return {"case": case, "logits": logits, "mask": mask, "aux_coef": 1e-3, "z_coef": 1e-3}
    if case["kind"] == "norm":
        T, H = case["rows"], case["width"]
        scale = torch.exp(_randn(gen, H, std=0.5))  # channels of unequal size, off centre
        return {"case": case, "x": (_randn(gen, T, H) * scale + 0.3).to(dt).requires_grad_(case["backward"]),
                "weight": (1.0 + _randn(gen, H, std=0.1)).requires_grad_(case["backward"]),
                "bias": _randn(gen, H, std=0.1).requires_grad_(case["backward"]), "eps": 1e-5,
                "grad": _randn(gen, T, H, dtype=dt)}
    if case["kind"] == "save8":
        T, H = case["rows"], case["width"]
        return {"case": case, "x": (_randn(gen, T, H) * torch.exp(_randn(gen, T, 1))).to(dt)}
    H, E, K, I = LAYERS[case["layer"]]
    T = case["tokens"]
    ids = torch.rand(T, E, generator=gen, device=DEV).topk(K, dim=1).indices
    w = torch.rand(T, K, generator=gen, device=DEV) + 0.1
    w = (w / w.sum(1, keepdim=True)).reshape(-1)
    # the pairs in expert order, as the permutation of the forward leaves them
    order = torch.sort(ids.reshape(-1), stable=True).indices
    inv_pos = torch.empty(T * K, dtype=torch.int32, device=DEV)
    inv_pos[order] = torch.arange(T * K, dtype=torch.int32, device=DEV)
    offs = torch.bincount(ids.reshape(-1), minlength=E).cumsum(0).to(torch.int32)
    return {"case": case, "hidden": _randn(gen, T, H, dtype=dt), "token": (order // K).to(torch.int32),
            "weight": w[order].contiguous(), "inv_pos": inv_pos, "offs": offs,
            "gate_up": _randn(gen, E, 2 * I, H, std=0.02, dtype=dt), "down": _randn(gen, E, H, I, std=0.02, dtype=dt),
            "grad": _randn(gen, T, H, dtype=dt)}


# ------------------------------------------------------------------ plain forms


def _plain_aux(st):
    logits, K = st["logits"], st["case"]["top_k"]
    lg = torch.stack([x.detach() for x in logits]).float()
    L, N, E = lg.shape
    m = torch.ones(N, 1, device=DEV) if st["mask"] is None else st["mask"].float()[:, None]
    n = m.sum() * L
    picked = torch.sort(lg, dim=-1, descending=True, stable=True).indices[..., :K]
    counts = (torch.zeros_like(lg).scatter_(2, picked, 1.0) * m).sum(1)
    top = lg.amax(-1, keepdim=True)
    ex = torch.exp(lg - top)
    tot = ex.sum(-1, keepdim=True)
    p, lse = ex / tot, top + torch.log(tot)
    total = counts.sum(0, dtype=torch.float64)
    psum = (p * m).sum((0, 1), dtype=torch.float64)
    one = n.clamp(min=1.0)
    balance = (E * (total / one) * (psum / one)).sum()
    z = (lse.square() * m).sum(dtype=torch.float64) / one
    f = ((total * E - K * n) / (one * E)).float()  # c / n less its mean K / E: the softmax's sum is one
    g = p * (st["aux_coef"] * E * (f - (p * f).sum(-1, keepdim=True)) + 2.0 * st["z_coef"] * lse) * (m / one)
    loss = st["aux_coef"] * balance + st["z_coef"] * z
    return {"loss": loss.float(), "load_balance": balance.float(), "z_loss": z.float(),
            "counts": counts.to(torch.int32), "grads": list(g.to(logits[0].dtype).unbind(0))}


def _plain_norm(st):
    x, w, b = st["x"].detach().float(), st["weight"].detach(), st["bias"].detach()
    xc = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(xc.square().mean(-1, keepdim=True) + st["eps"])
    xh = xc * r
    out = {"y": (xh * w + b).to(st["x"].dtype)}
    if st["case"]["backward"]:
        g = st["grad"].float()
        gw = g * w
        gx = r * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
        out |= {"grad_x": gx.to(st["x"].dtype), "grad_weight": (g * xh).sum(0), "grad_bias": g.sum(0)}
    return out


def _pow2(e):
    """2^e in 32 bits, from its bits, for e in [-126, 127]."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _through8(x, dt):
    """``x`` (fp32 values of type ``dt``) as its 8-bit checkpoint stands for it: per group of 32
    columns the least power of two whose codes reach at most 127; what is not finite becomes NaN."""
    C = x.shape[-1]
    v = torch.nn.functional.pad(x, (0, -C % GROUP)).unflatten(-1, (-1, GROUP))
    fine = torch.isfinite(v)
    a = torch.where(fine, v.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.frexp(a).exponent - 7  # a 2^-e in [64, 128)
    e = torch.where(a == 0, -126, e).clamp(min=-126)
    e = torch.where(a * _pow2(-e) >= 127.5, e + 1, e)
    q = torch.round(v * _pow2(-e))
    big = torch.finfo(dt).max
    v = torch.where(fine, (q * _pow2(e)).clamp(-big, big), math.nan)
    return v.flatten(-2)[..., :C]


def _plain_ffn8(st):
    """All experts' products as one batched product over rows padded to the fullest expert's."""
    dt, offs, token = st["hidden"].dtype, st["offs"].long(), st["token"].long()
    H, E, K, I = LAYERS[st["case"]["layer"]]
    row = torch.arange(token.numel(), device=DEV)
    expert = torch.searchsorted(offs, row, right=True)
    start = torch.cat([offs.new_zeros(1), offs[:-1]])
    slot = row - start[expert]
    cap = int((offs - start).max())
    down = st["down"].float()

    def spread(rows):  # the sorted pairs' rows -> (E, cap, .)
        return torch.zeros(E, cap, rows.shape[-1], device=DEV).index_put_((expert, slot), rows)

    w = st["weight"][:, None]
    gu = torch.bmm(spread(st["hidden"].float()[token]), st["gate_up"].float().transpose(1, 2).contiguous())
    gu = gu[expert, slot].to(dt).float()  # held in the inputs' type
    g, u = gu[:, :I], gu[:, I:]
    mid = g / (1.0 + torch.exp(-g)) * u * w
    gm = torch.bmm(spread(st["grad"].float()[token]), down)[expert, slot]
    g, u = _through8(g, dt), _through8(u, dt)
    s = 1.0 / (1.0 + torch.exp(-g))
    act = g * s * u
    dm = gm * w
    ggu = torch.cat([dm * u * s * (1.0 + g * (1.0 - s)), dm * g * s], -1)
    return {"mid": mid.to(dt), "mid_again": (act * w).to(dt), "grad_gate_up_out": ggu.to(dt),
            "grad_weights": (gm * act).sum(-1)[st["inv_pos"].long()].view(-1, K).to(dt)}


# --------------------------------------------------------------------- one pass


def run(state):
    kind = state["case"]["kind"]
    if own:
        import pluggy_amd
        from pluggy_amd import ops

        if kind == "aux":
            c = state["case"]
            r = pluggy_amd.router_aux_loss(state["logits"], c["experts"], c["top_k"], state["aux_coef"],
                                           state["z_coef"], token_mask=state["mask"])
            grads = torch.autograd.grad(r.loss, state["logits"])
            return {"loss": r.loss, "load_balance": r.load_balance, "z_loss": r.z_loss, "counts": r.expert_counts,
                    "grads": list(grads)}
        if kind == "norm":
            y = pluggy_amd.layer_norm(state["x"], state["weight"], state["bias"], state["eps"])
            if not state["case"]["backward"]:
                return {"y": y}
            gx, gw, gb = torch.autograd.grad(y, [state["x"], state["weight"], state["bias"]], state["grad"])
            return {"y": y, "grad_x": gx, "grad_weight": gw, "grad_bias": gb}
        if kind == "save8":
            codes, exps = ops.act8_save(state["x"])
            return {"x": ops.act8_restore(codes, exps, state["x"].dtype)}
        codes, exps, mid = ops.gate_up_swiglu_act8(state["hidden"], state["gate_up"], state["offs"], state["token"],
                                                   state["weight"])
        ggu, again, part = ops.down_proj_dgrad_act8(state["grad"], codes, exps, state["down"], state["offs"],
                                                    state["token"], state["weight"], need_part=True)
        gw = ops.pair_weight_grad(part, state["inv_pos"], LAYERS[state["case"]["layer"]][2], state["hidden"].dtype)
        return {"mid": mid, "mid_again": again, "grad_gate_up_out": ggu, "grad_weights": gw}
    if kind == "aux":
        return _plain_aux(state)
    if kind == "norm":
        return _plain_norm(state)
    if kind == "save8":
        return {"x": _through8(state["x"].float(), state["x"].dtype).to(state["x"].dtype)}
    return _plain_ffn8(state)


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "aux":  # logits in, gradients out
        n = case["layers"] * case["tokens"] * case["experts"]
        return {"bytes": 2 * n * es, "flops": 20 * n}
    if case["kind"] == "norm":  # x (and the gradient) in, y (and x's gradient) out
        n = case["rows"] * case["width"]
        return {"bytes": n * es * (4 if case["backward"] else 2) + case["width"] * (16 if case["backward"] else 8),
                "flops": n * (20 if case["backward"] else 8)}
    if case["kind"] == "save8":  # x in, the checkpoint out and in, x out
        n = case["rows"] * case["width"]
        return {"bytes": 2 * n * es + 2 * (n + n // GROUP), "flops": 6 * n}
    H, E, K, I = LAYERS[case["layer"]]
    P = case["tokens"] * K
    # hidden and grad in, both expert weights in, the checkpoint out and in, mid twice and the gradient out
    return {"bytes": es * (2 * case["tokens"] * H + 3 * E * H * I + 4 * P * I) + 2 * (2 * P * I + 2 * P * I // GROUP),
            "flops": 6 * P * H * I}


# ------------------------------------------------------------ results in 64 bits


def _exact_aux(st):
    K, E = st["case"]["top_k"], st["case"]["experts"]
    L, N = len(st["logits"]), st["case"]["tokens"]
    valid = torch.ones(N, dtype=torch.bool, device=DEV) if st["mask"] is None else st["mask"]
    n = int(valid.sum()) * L
    probs, lses, counts = [], [], []
    lower = torch.ones(E, E, dtype=torch.bool, device=DEV).tril(-1)  # [j, i]: i < j
    for lg in st["logits"]:
        l = lg.detach().double()
        hits = torch.zeros(E, dtype=torch.int64, device=DEV)
        for part, ok in zip(l.split(1024), valid.split(1024)):
            a, b = part[:, :, None], part[:, None, :]
            before = ((b > a) | ((b == a) & lower)).sum(-1)  # experts that rank ahead of j
            hits += ((before < K) & ok[:, None]).sum(0)
        counts.append(hits)
        lses.append(torch.logsumexp(l, -1))
        probs.append(torch.softmax(l, -1))
    total = torch.stack(counts).sum(0).double()
    f = total / max(n, 1)
    P = sum((p * valid[:, None]).sum(0) for p in probs) / max(n, 1)
    balance, z = E * (f * P).sum(), sum((s * s)[valid].sum() for s in lses) / max(n, 1)
    a, c = st["aux_coef"] * E / max(n, 1), st["z_coef"] * 2 / max(n, 1)
    grads = [(a * p * (f - (p @ f)[:, None]) + c * s[:, None] * p) * valid[:, None] for p, s in zip(probs, lses)]
    return {"loss": st["aux_coef"] * balance + st["z_coef"] * z, "load_balance": balance, "z_loss": z,
            "counts": torch.stack(counts).to(torch.int32), "grads": grads}


def _exact_norm(st):
    x, w, b = (st[k].detach().double() for k in ("x", "weight", "bias"))
    var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
    sd = (var + st["eps"]).sqrt()
    xh = (x - mu) / sd
    out = {"y": xh * w + b}
    if st["case"]["backward"]:
        g = st["grad"].double()
        H = x.shape[1]
        gw = g * w
        gx = (H * gw - gw.sum(-1, keepdim=True) - xh * (gw * xh).sum(-1, keepdim=True)) / (H * sd)
        out |= {"grad_x": gx, "grad_weight": torch.einsum("th,th->h", g, xh), "grad_bias": g.sum(0)}
    return out


def _exact8(x, dt):
    """The checkpoint's values of a 64-bit tensor, group by group."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[-1], GROUP):
        v = x[..., lo:lo + GROUP]
        a = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0).abs().amax(-1, keepdim=True)
        # a = m 2^x with 1/2 <= m < 1: 2^(x - 7) takes a to [64, 128)
        x7 = torch.frexp(a.clamp(min=2.0 ** -120)).exponent.to(torch.int64) - 7
        step = ((x7 + 1023) << 52).view(torch.float64)
        step = torch.where(torch.round(a / step) > 127, 2 * step, step)
        r = torch.round(v / step) * step
        out[..., lo:lo + GROUP] = torch.where(torch.isfinite(v), r.clamp(-torch.finfo(dt).max, torch.finfo(dt).max), math.nan)
    return out


def _exact_ffn8(st):
    dt = st["hidden"].dtype
    ends = st["offs"].tolist()
    I, K = st["down"].shape[2], LAYERS[st["case"]["layer"]][2]
    P = st["token"].numel()
    mid, again = (torch.zeros(P, I, dtype=torch.float64, device=DEV) for _ in range(2))
    ggu = torch.zeros(P, 2 * I, dtype=torch.float64, device=DEV)
    gw = torch.zeros(P, dtype=torch.float64, device=DEV)
    for e, (lo, hi) in enumerate(zip([0] + ends, ends)):
        t, w = st["token"][lo:hi].long(), st["weight"][lo:hi, None].double()
        g, u = (st["hidden"][t].double() @ st["gate_up"][e].double().T).to(dt).double().chunk(2, -1)
        mid[lo:hi] = torch.sigmoid(g) * g * u * w
        g, u = _exact8(g, dt), _exact8(u, dt)
        s = torch.sigmoid(g)
        gm = st["grad"][t].double() @ st["down"][e].double()
        gw[lo:hi] = (gm * s * g * u).sum(-1)
        again[lo:hi] = s * g * u * w
        gm = gm * w
        ggu[lo:hi] = torch.cat([gm * u * (s + g * s * (1 - s)), gm * s * g], -1)
    return {"mid": mid, "mid_again": again, "grad_gate_up_out": ggu, "grad_weights": gw[st["inv_pos"].long()].view(-1, K)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "aux":
        return _exact_aux(st)
    if case["kind"] == "norm":
        return _exact_norm(st)
    if case["kind"] == "save8":
        return {"x": _exact8(st["x"].double(), st["x"].dtype)}
    return _exact_ffn8(st)
