"""GPU: activations saved in 8 bits, and the expert FFN's backward from them.

The format is exact arithmetic, so codes, exponents and restored values equal a
plain statement of it bit for bit. The products' results from a checkpoint are
held to the formulas in 64 bits on the restored values: with eps the type's, half a
step (eps / 2) for the rounding to it, and (H + 64) 2^-24 of the terms' magnitudes for the
fp32 sums over H.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._gpu_helpers import DEV, gen, ref_grouped, routing

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def plain_save(x):
    """codes and exps of a (..., C) tensor, in numpy's 64 bits."""
    a = x.detach().cpu().double().numpy()
    C = a.shape[-1]
    pad = np.zeros((*a.shape[:-1], -C % 32))
    v = np.concatenate([a, pad], -1).reshape(*a.shape[:-1], -1, 32)
    fine = np.isfinite(v)
    top = np.where(fine, np.abs(v), 0.0).max(-1)
    e = np.maximum(np.frexp(top)[1] - 7, -126)
    e = np.where(top == 0, -126, e)
    e = np.where(np.rint(np.ldexp(top, -e)) > 127, e + 1, e)
    with np.errstate(invalid="ignore"):
        q = np.where(fine, np.rint(np.ldexp(np.where(fine, v, 0.0), -e[..., None])), -128)
    codes = torch.from_numpy(q.astype(np.int8)).reshape(*a.shape[:-1], -1)[..., :C]
    return codes, torch.from_numpy((e + 127).astype(np.uint8))


def plain_restore(codes, exps, dt):
    c = codes.cpu().double()
    C = c.shape[-1]
    e = exps.cpu().to(torch.int32) - 127
    v = torch.ldexp(c, e.repeat_interleave(32, -1)[..., :C].double())
    big = torch.finfo(dt).max
    return torch.where(c == -128, float("nan"), v.clamp(-big, big)).to(dt)


def values(shape, dt, seed):
    """Rows of sizes from the smallest to the largest, with zeros, and groups that hold one value only."""
    g = gen(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    lo, hi = {"fp32": (-150, 128), "bf16": (-140, 128), "fp16": (-25, 16)}[dt]
    x = x * torch.ldexp(torch.ones(1, dtype=torch.float64), torch.randint(lo, hi, (*shape[:-1], 1), generator=g).double())
    x[torch.rand(shape, generator=g) < 0.1] = 0.0
    big = torch.finfo(DT[dt]).max
    return x.clamp(-big, big).to(DT[dt])


def same(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.isnan(), b.isnan()) and torch.equal(
        a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (5, 33), (1, 4096), (77, 64), (64, 200), (130, 1001),
                                   (2, 7, 40), (4099, 96)])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_format(shape, dt):
    from pluggy_amd import ops

    x = values(shape, dt, sum(shape))
    codes, exps = ops.act8_save(x.to(DEV))
    want_c, want_e = plain_save(x)
    assert torch.equal(codes.cpu(), want_c) and torch.equal(exps.cpu(), want_e)
    for out in DT.values():
        assert same(ops.act8_restore(codes, exps, out).cpu(), plain_restore(want_c, want_e, out))


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_borders(dt):
    """Where the exponent steps (127.5 of a step), ties to even, the type's extremes, zeros of both signs."""
    big, small = torch.finfo(DT[dt]).max, torch.finfo(DT[dt]).smallest_normal
    rows = [[127.0, 126.5, 0.5, 1.5, 2.5, -0.5], [127.25, 1.0, -1.0], [127.5, 1.0, 3.0], [128.0, 1.0, 3.0],
            [255.0, 254.0, 1.0], [254.5, 1.0], [big, -big, big / 2, 1.0], [-big], [small, -small, 0.0],
            [small / 2, small / 4], [0.0, -0.0], [1.0]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    from pluggy_amd import ops

    x = x.to(DT[dt])
    codes, exps = ops.act8_save(x.to(DEV))
    want_c, want_e = plain_save(x)
    assert torch.equal(codes.cpu(), want_c) and torch.equal(exps.cpu(), want_e)
    back = ops.act8_restore(codes, exps, DT[dt]).cpu()
    assert same(back, plain_restore(want_c, want_e, DT[dt])) and back.isfinite().all()


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_not_finite_values(dt):
    """They come back as NaN and leave their group as it was."""
    from pluggy_amd import ops

    x = torch.randn(8, 96, generator=gen(1)).to(DT[dt])
    clean = ops.act8_restore(*ops.act8_save(x.to(DEV)), DT[dt]).cpu()
    x[2, 40] = x[2, 41] = 0.0
    want = ops.act8_restore(*ops.act8_save(x.to(DEV)), DT[dt]).cpu()
    x[2, 40], x[2, 41] = float("inf"), float("nan")
    x[5, :32] = float("-inf")
    back = ops.act8_restore(*ops.act8_save(x.to(DEV)), DT[dt]).cpu()
    assert back[2, 40:42].isnan().all() and back[5, :32].isnan().all()
    want[2, 40:42] = back[2, 40:42]
    want[5, :32] = back[5, :32]
    assert same(back, want) and torch.equal(back[6], clean[6])


def test_error_bound_and_strides():
    from pluggy_amd import ops

    x = torch.randn(64, 320, generator=gen(2)).to(DEV)
    back = ops.act8_restore(*ops.act8_save(x), torch.float32)
    top = x.view(64, 10, 32).abs().amax(-1, keepdim=True)
    assert ((back - x).view(64, 10, 32).abs() <= top / 127).all()
    codes, exps = ops.act8_save(x.t().contiguous().t())
    assert torch.equal(ops.act8_restore(codes, exps, torch.float32), back)
    odd = torch.zeros(64 * 320 + 1, device=DEV)[1:].view(64, 320)
    odd.copy_(x)
    assert torch.equal(ops.act8_restore(*ops.act8_save(odd), torch.float32), back)
    assert ops.act8_save(torch.empty(0, 40, device=DEV))[1].shape == (0, 2)
    assert ops.act8_restore(*ops.act8_save(torch.empty(0, 40, device=DEV)), torch.float32).shape == (0, 40)


# ------------------------------------------------------- the expert products

# T, K, E, H, I: few rows an expert, half-filled tiles, 128- and 256-row tiles, odd widths, one expert
SHAPES = [(1, 1, 1, 8, 8), (3, 2, 4, 64, 24), (40, 2, 16, 128, 96), (257, 2, 4, 128, 72), (700, 4, 8, 256, 264),
          (1300, 2, 4, 512, 512), (64, 8, 64, 256, 768)]


def layer(T, K, E, H, I, dt, seed, mode="uniform", std=0.1):
    g = gen(seed)
    t = {"hidden": torch.randn(T, H, generator=g), "gate_up": torch.randn(E, 2 * I, H, generator=g) * std,
         "down": torch.randn(E, H, I, generator=g) * std, "grad": torch.randn(T, H, generator=g),
         "weights": torch.rand(T, K, generator=g) + 0.1}
    t = {k: v.to(DT[dt]).to(DEV) for k, v in t.items()}
    t["ids"] = routing(T, K, E, seed=seed, mode=mode).to(DEV)
    return t


@pytest.mark.parametrize("T,K,E,H,I", SHAPES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("mode", ["uniform", "zipf"])
def test_products_around_the_checkpoint(T, K, E, H, I, dt, mode):
    from pluggy_amd import ops

    t = layer(T, K, E, H, I, dt, T + I, mode)
    _, offs, _, inv_pos, tok, sw = ops.permute_rows(t["ids"], t["weights"], E)
    gu, mid = ops.gate_up_swiglu(t["hidden"], t["gate_up"], offs, tok, sw)
    codes, exps, mid8 = ops.gate_up_swiglu_act8(t["hidden"], t["gate_up"], offs, tok, sw)
    assert torch.equal(mid, mid8)
    P = T * K
    want_c, want_e = ops.act8_save(gu.view(P, 2, I))
    assert torch.equal(codes.view(P, 2, I), want_c) and torch.equal(exps, want_e)
    back = ops.act8_restore(want_c, want_e, DT[dt]).view(P, 2 * I)

    ggu, again, part = ops.down_proj_dgrad_act8(t["grad"], codes, exps, t["down"], offs, tok, sw, need_part=True)
    only, none, _ = ops.down_proj_dgrad_act8(t["grad"], codes, exps, t["down"], offs, tok, sw, need_mid=False)
    assert none is None and torch.equal(only, ggu)
    plain, plain_part = ops.down_proj_dgrad(t["grad"], back, t["down"], offs, tok, sw, need_part=True)
    assert torch.equal(ggu, plain) and torch.equal(part, plain_part)

    # the formulas in 64 bits on the restored values
    g, u = back.cpu().double().chunk(2, -1)
    s, w = torch.sigmoid(g), sw.cpu().double()[:, None]
    act = g * s * u
    half = 0.0 if dt == "fp32" else torch.finfo(DT[dt]).eps / 2
    tiny = torch.finfo(DT[dt]).smallest_normal * torch.finfo(DT[dt]).eps
    lim = (half + 32 * U) * (act * w).abs() + tiny
    assert ((again.cpu().double() - act * w).abs() <= lim).all()
    rows = t["grad"][tok.long()].cpu()
    gm = ref_grouped(rows, t["down"], offs, False)
    size = ref_grouped(rows.double().abs(), t["down"].double().abs(), offs, False)
    n = (H + 64) * U
    dg, du = u * s * (1 + g * (1 - s)) * w, g * s * w
    dsize = (u * s * (1 + g.abs() * (1 - s)) * w).abs()
    for got, want, lim in ((ggu[:, :I], gm * dg, (n + 32 * U) * size * dsize), (ggu[:, I:], gm * du, n * size * du.abs())):
        err = (got.cpu().double() - want).abs()
        lim = lim + 32 * U * want.abs() + half * (want.abs() + lim) + tiny
        assert (err <= lim).all(), (err / lim).max().item()
    gw = ops.pair_weight_grad(part, inv_pos, K).cpu().double().reshape(-1)
    want = (gm * act).sum(-1)[inv_pos.cpu().long()]
    lim = ((n + (I + 64) * U) * size * act.abs()).sum(-1)[inv_pos.cpu().long()]
    assert ((gw - want).abs() <= lim + tiny).all()


def test_without_row_weights_and_on_sorted_rows():
    from pluggy_amd import ops

    t = layer(200, 1, 4, 64, 40, "bf16", 3)
    _, offs, _, _, tok, _ = ops.permute_rows(t["ids"], t["weights"], 4)
    x, grad = t["hidden"][tok.long()], t["grad"][tok.long()]
    gu, mid = ops.gate_up_swiglu(x, t["gate_up"], offs)
    codes, exps, mid8 = ops.gate_up_swiglu_act8(x, t["gate_up"], offs)
    assert torch.equal(mid, mid8)
    back = ops.act8_restore(codes.view(200, 2, 40), exps, torch.bfloat16).view(200, 80)
    ggu, again, part = ops.down_proj_dgrad_act8(grad, codes, exps, t["down"], offs)
    assert part is None and torch.equal(ggu, ops.down_proj_dgrad(grad, back, t["down"], offs)[0])
    g, u = back.double().chunk(2, -1)
    want = g * torch.sigmoid(g) * u
    assert ((again.double() - want).abs() <= (2.0 ** -8 + 32 * U) * want.abs() + 1e-38).all()


def test_not_finite_preactivations_reach_the_gradient():
    """A gate that overflowed is NaN in the gradients of its row, as an unchecked block's would be not finite."""
    import pluggy_amd

    t = layer(40, 1, 2, 64, 32, "bf16", 4)
    t["hidden"][7, 3] = float("inf")
    x = t["hidden"].requires_grad_()
    out = pluggy_amd.moe_expert_ffn(x, t["ids"], t["weights"], t["gate_up"], t["down"], checkpoint_8bit=True)
    (gx,) = torch.autograd.grad(out, [x], t["grad"])
    assert gx[7].isnan().any() and gx[torch.arange(40) != 7].isfinite().all()


# --------------------------------------------------------------- the layer


def ffn_reference(t, gu, offs, tok, sw, inv_pos, dt):
    """Output and gradients in 64 bits from the saved pre-activations ``gu`` of the sorted rows: the output
    from gu itself, the gradients from its 8-bit checkpoint."""
    T, K = t["ids"].shape
    P, I = gu.shape[0], gu.shape[1] // 2
    E = t["gate_up"].shape[0]
    back = plain_restore(*plain_save(gu.view(P, 2, I)), dt).view(P, 2 * I)
    tok, inv, w = tok.cpu().long(), inv_pos.cpu().long(), sw.cpu().double()[:, None]

    def per_token(rows):
        return rows[inv].view(T, K, -1).sum(1)

    g, u = gu.cpu().double().chunk(2, -1)
    out = per_token(ref_grouped(g * torch.sigmoid(g) * u * w, t["down"].detach(), offs, True))
    g, u = back.double().chunk(2, -1)
    s = torch.sigmoid(g)
    rows = t["grad"].detach().cpu().double()[tok]
    gm = ref_grouped(rows, t["down"].detach(), offs, False)
    gw = (gm * g * s * u).sum(-1)[inv].view(T, K)
    ggu = torch.cat([gm * w * u * s * (1 + g * (1 - s)), gm * w * g * s], -1)
    gx = per_token(ref_grouped(ggu, t["gate_up"].detach(), offs, False))
    x = t["hidden"].detach().cpu().double()[tok]
    act = g * s * u * w
    ends = [0, *offs.tolist()]
    ggw = torch.stack([ggu[a:b].t() @ x[a:b] for a, b in zip(ends, ends[1:])])
    gdn = torch.stack([rows[a:b].t() @ act[a:b] for a, b in zip(ends, ends[1:])])
    return [out, gx, gw, ggw, gdn]


@pytest.mark.parametrize("T,K,E,H,I", [(1, 2, 4, 64, 32), (50, 2, 8, 64, 48), (300, 4, 8, 128, 96), (33, 2, 4, 60, 20)])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_expert_ffn_with_a_checkpoint(T, K, E, H, I, dt):
    """Output bit for bit the plain call's; gradients within the roundings of the types: at most six to ``dt``
    on the way to any of them, in the 2-norm."""
    import pluggy_amd
    from pluggy_amd import ops

    t = layer(T, K, E, H, I, dt, T + 1)
    leaves = [t[k].requires_grad_() for k in ("hidden", "weights", "gate_up", "down")]
    out = pluggy_amd.moe_expert_ffn(t["hidden"], t["ids"], t["weights"], t["gate_up"], t["down"], checkpoint_8bit=True)
    want = pluggy_amd.moe_expert_ffn(t["hidden"], t["ids"], t["weights"], t["gate_up"], t["down"])
    assert torch.equal(out, want)
    grads = torch.autograd.grad(out, leaves, t["grad"])
    if H % 8 or I % 8:  # padded on the way in: compared with the exact backward below the checkpoint's error
        exact = torch.autograd.grad(want, leaves, t["grad"])
        for a, b in zip(grads, exact):
            assert (a - b).float().norm() <= 0.05 * b.float().norm()
        return
    _, offs, _, inv_pos, tok, sw = ops.permute_rows(t["ids"], t["weights"].detach(), E)
    gu, _ = ops.gate_up_swiglu(t["hidden"].detach(), t["gate_up"].detach(), offs, tok, sw)
    ref = ffn_reference(t, gu, offs, tok, sw, inv_pos, DT[dt])
    tol = 6 * (torch.finfo(DT[dt]).eps / 2) + 4 * (H + 2 * I + T * K + 64) * U
    for got, r in zip((out.detach(), *grads), ref):
        rel = (got.cpu().double() - r).norm() / r.norm()
        assert rel <= tol, (rel.item(), tol)


@pytest.mark.parametrize("needs", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_only_the_wanted_gradients(needs):
    import pluggy_amd

    t = layer(60, 2, 4, 64, 32, "bf16", 5)
    names = ("hidden", "weights", "gate_up", "down")
    full = [t[k].clone().requires_grad_() for k in names]
    part = [t[k].clone().requires_grad_(i in needs) for i, k in enumerate(names)]

    def grads(p, which):
        out = pluggy_amd.moe_expert_ffn(p[0], t["ids"], p[1], p[2], p[3], checkpoint_8bit=True)
        return torch.autograd.grad(out, [p[i] for i in which], t["grad"])

    for a, b in zip(grads(part, needs), [grads(full, range(4))[i] for i in needs]):
        assert torch.equal(a, b)


def build_mlp(H=64, I=32, E=8, K=2, dtype=torch.float32, seed=0):
    import pluggy_amd

    torch.manual_seed(seed)
    mlp = pluggy_amd.Qwen3MoeSparseMLP(H, I, E, K).to(DEV)
    for p in mlp.parameters():
        torch.nn.init.normal_(p, std=0.2)
    return mlp.to(dtype)


@pytest.mark.parametrize("path", ["mlp", "sublayer", "experts", "layernorm"])
@pytest.mark.parametrize("amp", [False, True])
def test_modules_keep_8_bits(path, amp):
    """Every path of the modules: output and statistics unchanged, less kept, gradients near the exact ones
    (each of the pre-activations off by at most 1/127 of its group's largest: within 5 % in the norm)."""
    import pluggy_amd

    mlp = build_mlp()
    norm = (torch.nn.LayerNorm if path == "layernorm" else torch.nn.RMSNorm)(64).to(DEV)
    x = torch.randn(2, 37, 64, generator=gen(6)).to(DEV)
    got = []
    for flag in (False, True):
        mlp.experts.checkpoint_8bit = flag
        xi = x.clone().requires_grad_()
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t), \
                torch.autocast("cuda", torch.bfloat16, enabled=amp):
            if path == "mlp":
                y = mlp(xi)
            elif path == "experts":
                _, w, idx = mlp.router(xi.view(-1, 64))
                y = mlp.experts(xi.view(-1, 64), idx, w).view(2, 37, 64)
            else:
                y = pluggy_amd.moe_sublayer(xi, norm, mlp)
        params = [xi, *mlp.parameters()] + ([] if path in ("mlp", "experts") else list(norm.parameters()))
        grads = torch.autograd.grad(y, params, torch.ones_like(y))
        got.append((y, grads, {t.dtype for t in kept}))
    assert torch.equal(got[0][0], got[1][0])
    assert torch.int8 in got[1][2] and torch.int8 not in got[0][2]
    for a, b in zip(got[0][1], got[1][1]):
        assert (a - b).norm() <= 0.05 * a.norm() and a.norm() > 0


def test_no_rows_and_no_gradient():
    mlp = build_mlp(dtype=torch.bfloat16)
    mlp.experts.checkpoint_8bit = True
    x = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = mlp(x)
    grads = torch.autograd.grad(y, [x, *mlp.parameters()], torch.empty_like(y))
    assert grads[0].shape == x.shape and not any(g.any() for g in grads[1:])
    x = torch.randn(1, 9, 64, device=DEV).bfloat16()
    with torch.no_grad():
        a = mlp(x)
        mlp.experts.checkpoint_8bit = False
        assert torch.equal(a, mlp(x))


def test_two_backwards_of_one_forward():
    import pluggy_amd

    t = layer(80, 2, 4, 64, 32, "bf16", 7)
    x = t["hidden"].requires_grad_()
    out = pluggy_amd.moe_expert_ffn(x, t["ids"], t["weights"], t["gate_up"], t["down"], checkpoint_8bit=True)
    a = torch.autograd.grad(out, [x], t["grad"], retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(out, [x], t["grad"])[0])


def test_compiled_matches_eager():
    mlp = build_mlp(dtype=torch.bfloat16)
    mlp.experts.checkpoint_8bit = True
    x = torch.randn(1, 40, 64, generator=gen(8)).bfloat16().to(DEV).requires_grad_()
    params = [x, *mlp.parameters()]
    y = mlp(x)
    yc = torch.compile(mlp, backend="aot_eager")(x)
    assert torch.equal(y, yc)
    g = torch.ones_like(y)
    for a, b in zip(torch.autograd.grad(y, params, g), torch.autograd.grad(yc, params, g)):
        assert torch.equal(a, b)


def test_backward_under_capture_raises(monkeypatch):
    import pluggy_amd

    t = layer(20, 2, 4, 64, 32, "bf16", 9)
    x = t["hidden"].requires_grad_()
    out = pluggy_amd.moe_expert_ffn(x, t["ids"], t["weights"], t["gate_up"], t["down"], checkpoint_8bit=True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="not supported under HIP graph capture"):
        torch.autograd.grad(out, [x], t["grad"])


def test_a_training_step_of_all_together():
    """LayerNorm, router with its auxiliary loss, experts with an 8-bit checkpoint: one step's gradients
    against the same step on exact activations, and the auxiliary loss's own share against its torch form."""
    import pluggy_amd

    H, E, K, T = 64, 8, 2, 45
    x = torch.randn(1, T, H, generator=gen(10)).to(DEV)
    mask = torch.arange(T, device=DEV) < 40
    got = []
    for flag in (False, True):
        mlps = [build_mlp(seed=i) for i in range(2)]
        norms = [torch.nn.LayerNorm(H).to(DEV) for _ in mlps]
        h = x
        for m, norm in zip(mlps, norms):
            m.experts.checkpoint_8bit = flag
            h = pluggy_amd.moe_sublayer(h, norm, m)
        aux = pluggy_amd.router_aux_loss([m.last_router_logits for m in mlps], E, K, 0.1, 0.01, token_mask=mask)
        loss = h.square().mean() + aux.loss
        params = [p for m, n in zip(mlps, norms) for p in (*m.parameters(), *n.parameters())]
        got.append((loss.detach(), torch.autograd.grad(loss, params), aux.expert_counts))
        assert aux.expert_counts.sum().item() == 2 * 40 * K
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][2], got[1][2])
    for a, b in zip(got[0][1], got[1][1]):
        assert (a - b).norm() <= 0.05 * a.norm() and a.norm() > 0


def test_in_a_graph_and_on_another_stream():
    """Saving, restoring and the GEMMs around the checkpoint, replayed on changed inputs with eager work between."""
    import pluggy_amd
    from pluggy_amd import ops

    mlp = pluggy_amd.Qwen3MoeSparseMLP(64, 48, 8, 2).to(DEV).to(torch.bfloat16)
    mlp.experts.checkpoint_8bit = True
    g = gen(91)
    with torch.no_grad():
        for p in mlp.parameters():
            p.copy_((torch.randn(p.shape, generator=g) * 0.1).to(DEV))
    x = torch.randn(1, 300, 64, generator=g).to(torch.bfloat16).to(DEV)

    def step():
        codes, exps = ops.act8_save(x)
        return ops.act8_restore(codes, exps, torch.bfloat16), codes, exps, mlp(x).detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.mul_(1.5)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


def test_past_32_bit_offsets():
    """2.2e9 values: the last rows are those of the rows by themselves."""
    from pluggy_amd import ops

    R, C = 1100000, 2000
    x = torch.randn(R, C, device=DEV, dtype=torch.bfloat16)
    codes, exps = ops.act8_save(x)
    back = ops.act8_restore(codes, exps, torch.bfloat16)
    for rows in (slice(0, 40), slice(R - 40, R)):
        c, e = ops.act8_save(x[rows])
        assert torch.equal(codes[rows], c) and torch.equal(exps[rows], e)
        assert torch.equal(back[rows], ops.act8_restore(c, e, torch.bfloat16))
