"""GPU: the router's auxiliary loss, its counts and gradients against the formulas in 64 bits.

Bounds, with u = 2^-24: a probability is one expf (2 u, and its argument's
rounding, |x - max| u <= 40 u for the logits here), a sum of at most 1024 of them in a
tree of depth 16 + 6, a division: 72 u in all relative; a gradient has a few more operations on terms of
its size: 96 u of sum of the terms' magnitudes, and half a step of the logits' type. The sums over rows
are of positive terms: 128 more steps cover a thread's rows and the joins.
"""

from __future__ import annotations

import pytest
import torch

from tests._gpu_helpers import DEV, gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def select(l, K):
    """(N, E) truth values of the K largest, equal ones by id."""
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :K]
    return torch.zeros_like(l, dtype=torch.bool).scatter_(1, order, True)


def reference(logits, K, a, z, mask=None, gscale=1.0):
    E = logits[0].shape[1]
    keep = [torch.ones(l.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1) != 0 for l in logits]
    ls = [l.detach().cpu().double() for l in logits]
    picks = [select(l, K) & k[:, None] for l, k in zip(ls, keep)]
    counts = torch.stack([p.sum(0) for p in picks])
    n = sum(int(k.sum()) for k in keep)
    probs = [torch.softmax(l, -1) for l in ls]
    lses = [torch.logsumexp(l, -1) for l in ls]
    if n == 0:
        return {"loss": 0.0, "lb": 0.0, "z": 0.0, "counts": counts, "grads": [torch.zeros_like(l) for l in ls],
                "bounds": [torch.zeros_like(l) for l in ls]}
    f = counts.sum(0).double() / n
    P = sum(p[k].sum(0) for p, k in zip(probs, keep)) / n
    lb, zl = E * (f * P).sum(), sum(s[k].square().sum() for s, k in zip(lses, keep)) / n
    fc = f - K / E
    grads, bounds = [], []
    for p, s, k in zip(probs, lses, keep):
        m = (p @ fc)[:, None]
        g = gscale * p / n * (a * E * (fc - m) + 2 * z * s[:, None])
        b = abs(gscale) * p / n * (a * E * (fc.abs() + (p @ fc.abs())[:, None]) + 2 * z * (s.abs()[:, None] + 1))
        grads.append(torch.where(k[:, None], g, 0.0))
        bounds.append(96 * U * torch.where(k[:, None], b, 0.0))
    return {"loss": float(a * lb + z * zl), "lb": float(lb), "z": float(zl), "counts": counts, "grads": grads,
            "bounds": bounds}


def check(r, grads, ref, a, z):
    assert torch.equal(r.expert_counts.cpu().long(), ref["counts"])
    assert r.expert_counts.dtype == torch.int32
    tol = 256 * U
    for got, want, size in ((r.load_balance, ref["lb"], ref["lb"]), (r.z_loss, ref["z"], ref["z"]),
                            (r.loss, ref["loss"], a * ref["lb"] + z * ref["z"])):
        assert got.dtype == torch.float32 and got.shape == ()
        assert abs(got.item() - want) <= tol * abs(size), (got.item(), want)
    for g, want, bound in zip(grads, ref["grads"], ref["bounds"]):
        dt = g.dtype
        half = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
        lim = bound + (want.abs() + bound) * half + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        err = (g.cpu().double() - want).abs()
        assert (err <= lim).all(), (err / lim).max().item()


def draw(L, N, E, dt, seed, spread=1.0):
    g = gen(seed)
    return [((torch.randn(N, E, generator=g) + 0.5 * torch.randn(E, generator=g)) * spread).to(DT[dt]).to(DEV)
            .requires_grad_() for _ in range(L)]


def run(logits, K, a, z, mask=None, gscale=1.0, **kw):
    import pluggy_amd

    r = pluggy_amd.router_aux_loss(logits, logits[0].shape[1], K, a, z, token_mask=mask, **kw)
    return r, torch.autograd.grad(r.loss * gscale, logits)


@pytest.mark.parametrize("E,K", [(1, 1), (2, 1), (3, 3), (4, 2), (16, 4), (17, 5), (32, 4), (33, 8), (60, 6), (64, 8),
                                 (100, 7), (128, 8), (130, 8), (256, 10), (300, 16), (512, 64), (513, 2), (1024, 64)])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_experts_and_types(E, K, dt):
    logits = draw(2, 77, E, dt, E * 7 + K)
    gscale = 512.0  # keeps fp16 gradients above its smallest steps
    r, grads = run(logits, K, 1e-2, 1e-3, gscale=gscale)
    check(r, grads, reference(logits, K, 1e-2, 1e-3, gscale=gscale), 1e-2, 1e-3)


@pytest.mark.parametrize("L,N", [(1, 1), (1, 2), (1, 63), (3, 64), (1, 4097), (12, 513), (48, 100), (64, 9), (65, 9),
                                 (130, 5)])
@pytest.mark.parametrize("masked", [False, True])
def test_layers_rows_and_masks(L, N, masked):
    logits = draw(L, N, 32, "fp32", L + N)
    mask = (torch.rand(N, generator=gen(N)) < 0.6).to(DEV) if masked else None
    r, grads = run(logits, 4, 1e-3, 1e-3, mask)
    check(r, grads, reference(logits, 4, 1e-3, 1e-3, mask), 1e-3, 1e-3)


def test_layers_of_unlike_rows():
    g = gen(3)
    logits = [torch.randn(n, 24, generator=g).to(DEV).requires_grad_() for n in (5, 0, 700, 64)]
    r, grads = run(logits, 3, 0.5, 0.25)
    check(r, grads, reference(logits, 3, 0.5, 0.25), 0.5, 0.25)
    assert grads[1].shape == (0, 24)


@pytest.mark.parametrize("a,z", [(1.0, 0.0), (0.0, 1.0), (0.0, 0.0), (-1.0, 2.0)])
def test_coefficients(a, z):
    logits = draw(2, 50, 16, "fp32", 4)
    r, grads = run(logits, 2, a, z)
    ref = reference(logits, 2, a, z)
    ref["bounds"] = reference(logits, 2, abs(a), abs(z))["bounds"]
    check(r, grads, ref, abs(a), abs(z))


@pytest.mark.parametrize("E,K", [(8, 3), (32, 4), (128, 8), (130, 64), (1024, 5)])
@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_ties_go_to_the_lower_id(E, K, dt):
    """All logits equal (a zero-initialised router), few distinct values, and zeros of both signs."""
    g = gen(E)
    same = torch.zeros(40, E)
    few = torch.randint(0, 3, (40, E), generator=g).float()
    signs = torch.where(torch.rand(40, E, generator=g) < 0.5, 0.0, -0.0)
    logits = [t.to(DT[dt]).to(DEV).requires_grad_() for t in (same, few, signs)]
    r, grads = run(logits, K, 1.0, 0.1)
    check(r, grads, reference([t.abs() if i == 2 else t for i, t in enumerate(logits)], K, 1.0, 0.1), 1.0, 0.1)
    assert r.expert_counts[0, :K].eq(40).all() and r.expert_counts[0, K:].eq(0).all()
    assert torch.equal(r.expert_counts[0], r.expert_counts[2])


def test_a_balanced_router_keeps_its_gradient():
    """Counts within one of each other: f_j - sum f p is a small difference, and keeps its digits."""
    N, E, K = 4096, 64, 2
    base = torch.randn(N, E, generator=gen(5)) * 0.01
    base[torch.arange(N), torch.arange(N) % E] += 1.0
    base[torch.arange(N), (torch.arange(N) + 1) % E] += 1.0
    base[0, :3] = torch.tensor([0.0, 5.0, 5.0])  # a pair out of order
    logits = [base.to(DEV).requires_grad_()]
    r, grads = run(logits, K, 1.0, 0.0)
    ref = reference(logits, K, 1.0, 0.0)
    check(r, grads, ref, 1.0, 0.0)
    rel = (grads[0].cpu().double() - ref["grads"][0]).norm() / ref["grads"][0].norm()
    assert rel < 96 * U


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min])
def test_masked_rows_may_hold_anything(fill):
    logits = draw(2, 90, 40, "fp32", 6)
    mask = torch.ones(90, dtype=torch.bool, device=DEV)
    mask[::3] = False
    want, gwant = run(logits, 4, 1e-2, 1e-2, mask)
    dirty = [torch.where(mask[:, None], l.detach(), fill).requires_grad_() for l in logits]
    got, grads = run(dirty, 4, 1e-2, 1e-2, mask)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.expert_counts, want.expert_counts)
    for g, w in zip(grads, gwant):
        assert torch.equal(g, w) and not g[::3].any()


def test_no_row_left():
    logits = draw(2, 30, 16, "bf16", 7)
    r, grads = run(logits, 2, 1.0, 1.0, torch.zeros(30, dtype=torch.bool, device=DEV))
    assert r.loss.item() == r.load_balance.item() == r.z_loss.item() == 0.0
    assert not r.expert_counts.any() and not any(g.any() for g in grads)
    none = [torch.empty(0, 16, device=DEV, requires_grad=True)]
    r, grads = run(none, 2, 1.0, 1.0)
    assert r.loss.item() == 0.0 and grads[0].shape == (0, 16)


def test_masks_of_other_types_and_shapes():
    logits = draw(2, 24, 8, "fp32", 8)
    mask = torch.rand(4, 6, generator=gen(8)) < 0.5
    want, gwant = run(logits, 2, 1.0, 1.0, mask.to(DEV))
    for m in (mask.long(), mask.to(torch.uint8) * 3, mask.int(), mask.t().contiguous().t()):
        got, grads = run(logits, 2, 1.0, 1.0, m.to(DEV))
        assert torch.equal(got.loss, want.loss) and all(torch.equal(g, w) for g, w in zip(grads, gwant))


def test_values_below_the_masking_one():
    """Experts masked out with -inf or the type's lowest value have no probability and no gradient."""
    for low in (float("-inf"), torch.finfo(torch.float32).min):
        base = torch.randn(50, 16, generator=gen(9))
        base[:, 3] = base[:, 11] = low
        logits = [base.to(DEV).requires_grad_()]
        r, grads = run(logits, 4, 1.0, 1.0)
        ref = reference(logits, 4, 1.0, 1.0)
        assert torch.equal(r.expert_counts.cpu().long(), ref["counts"]) and not r.expert_counts[0, 3].any()
        check(r, grads, ref, 1.0, 1.0)
        assert not grads[0][:, 3].any()


def test_not_finite_logits_give_nan():
    for bad in (float("nan"), float("inf")):
        logits = draw(1, 20, 16, "fp32", 10)
        with torch.no_grad():
            logits[0][5, 7] = bad
        r, grads = run(logits, 2, 1.0, 1.0)
        assert r.loss.isnan() and grads[0][5].isnan().all()
        assert torch.equal(r.expert_counts.cpu().long(), reference(logits, 2, 1.0, 1.0)["counts"])


def test_strided_and_unaligned_logits():
    wide = torch.randn(60, 41, generator=gen(11)).to(DEV)
    flat = torch.randn(60 * 32 + 3, generator=gen(12)).to(DEV)
    views = [wide[:, 5:37], wide.t()[3:35].t(), flat[1:1 + 60 * 32].view(60, 32), flat[3:].view(60, 32)]
    logits = [v.detach().requires_grad_() for v in views]
    r, grads = run(logits, 4, 1e-2, 1e-2)
    check(r, grads, reference(logits, 4, 1e-2, 1e-2), 1e-2, 1e-2)


def test_unaligned_16_bit_rows():
    """Rows of 8 and of 2 bytes' alignment, and gradients of some layers only."""
    for E in (60, 61):
        logits = draw(3, 101, E, "bf16", E)
        import pluggy_amd

        r = pluggy_amd.router_aux_loss(logits, E, 6, 1.0, 0.1)
        ref = reference(logits, 6, 1.0, 0.1)
        for which in ([0, 2], [1]):
            got = torch.autograd.grad(r.loss, [logits[i] for i in which], retain_graph=True)
            check(r, got, {**ref, "grads": [ref["grads"][i] for i in which],
                           "bounds": [ref["bounds"][i] for i in which]}, 1.0, 0.1)


def test_gradient_matches_differences():
    """Along a direction, at logits whose order does not change: the counts are then constants."""
    logits = draw(2, 30, 12, "fp32", 13)
    r, grads = run(logits, 3, 1.0, 0.5)
    ds = [torch.randn(l.shape, generator=gen(14), dtype=torch.float64) for l in logits]
    c = r.expert_counts.cpu().double().sum(0)

    def loss(h):
        ls = [l.detach().cpu().double() + h * d for l, d in zip(logits, ds)]
        n = sum(len(l) for l in ls)
        P = sum(torch.softmax(l, -1).sum(0) for l in ls) / n
        return 12 * (c / n * P).sum() + 0.5 * sum(torch.logsumexp(l, -1).square().sum() for l in ls) / n

    h = 1e-5
    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((g.cpu().double() * d).sum() for g, d in zip(grads, ds))
    scale = sum((g.cpu().double().abs() * d.abs()).sum() for g, d in zip(grads, ds))
    assert abs(got - want) <= (200 * U + 1e-8) * scale


def test_matches_the_framework_and_follows_its_statistics():
    """From the logits and from the fused routers' statistics, against the torch forms beside it."""
    import pluggy_amd

    T, H, E, K = 512, 64, 32, 4
    layers = []
    for i in range(3):
        x = torch.randn(T, H, generator=gen(20 + i)).to(DEV)
        w = (torch.randn(E, H, generator=gen(30 + i)) * 0.2).to(DEV)
        logits, _, _, stats = pluggy_amd.router_topk(x, w, K, return_stats=True)
        layers.append((logits.detach().requires_grad_(), stats))
    logits, stats = [l for l, _ in layers], [s for _, s in layers]
    lb = pluggy_amd.load_balancing_loss(logits, E, K)
    zl = torch.logsumexp(torch.cat(logits), -1).square().mean()
    want = torch.autograd.grad(0.3 * lb + 0.2 * zl, logits)
    ref = reference(logits, K, 0.3, 0.2)
    for kw in ({}, {"stats": stats}):
        r, grads = run(logits, K, 0.3, 0.2, **kw)
        check(r, grads, ref, 0.3, 0.2)
        assert torch.equal(r.expert_counts, torch.stack([s.expert_counts for s in stats]))
        torch.testing.assert_close(r.load_balance, lb.detach(), rtol=512 * U, atol=0)
        for g, w in zip(grads, want):
            torch.testing.assert_close(g, w, rtol=1e-3, atol=1e-9)


def test_many_layers_from_statistics():
    import pluggy_amd
    from pluggy_amd import RouterStats

    logits = draw(70, 40, 20, "fp32", 15)
    stats = []
    for l in logits:
        d = l.detach().double()
        stats.append(RouterStats(select(l.detach(), 3).sum(0).int(), torch.softmax(d, -1).sum(0).float(),
                                 torch.logsumexp(d, -1).square().sum().float().reshape(1), 40))
    r, grads = run(logits, 3, 1.0, 1.0, stats=stats)
    check(r, grads, reference(logits, 3, 1.0, 1.0), 1.0, 1.0)
    assert pluggy_amd.router_aux_loss([], 20, 3).loss.item() == 0.0


def test_install_stats_aux_fused():
    """The reference model's hook with ``fused``: the loss and the gradients of every router of the torch form."""
    import types

    import pluggy_amd

    def model():
        torch.manual_seed(1)
        blocks = []
        for _ in range(2):
            mlp = pluggy_amd.Qwen3MoeSparseMLP(32, 16, 8, 2).to(DEV)
            for p in mlp.parameters():
                torch.nn.init.normal_(p, std=0.3)
            blocks.append(types.SimpleNamespace(ffn=mlp))
        return types.SimpleNamespace(blocks=blocks, num_experts=8, router_aux_loss_coef=0.1, router_z_loss_coef=0.2)

    got = []
    for fused in (False, True):
        m = model()
        pluggy_amd.install_stats_aux(m, fused=fused)
        x = torch.randn(2, 21, 32, generator=gen(16)).to(DEV)
        for b in m.blocks:
            b.ffn(x)
        m._router_logits = [b.ffn.last_router_logits for b in m.blocks]
        loss = m.aux_loss()
        got.append([loss.detach(), *torch.autograd.grad(loss, [b.ffn.router.weight for b in m.blocks])])
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-7)


def test_deterministic_and_on_another_stream():
    logits = draw(12, 4000, 64, "fp32", 17)
    r, grads = run(logits, 6, 1e-3, 1e-3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r2, grads2 = run(logits, 6, 1e-3, 1e-3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(r.loss, r2.loss) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_losses_can_be_changed_in_place():
    logits = draw(1, 20, 8, "fp32", 18)
    import pluggy_amd

    r = pluggy_amd.router_aux_loss(logits, 8, 2, 1.0, 1.0)
    total = r.loss
    total += 1.0
    total.backward()
    assert logits[0].grad is not None


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
def test_values_far_apart_and_close_together(dt):
    """Rows whose maximum is so far above the rest that differences from it lose digits (equal after the
    subtraction, not before), rows of neighbours in the type, and infinities on both ends of the order."""
    E, K = 48, 5
    g = gen(21)
    eps = torch.finfo(DT[dt]).eps
    far = torch.randn(60, E, generator=g) * 1e-3
    far[torch.arange(60), torch.randint(0, E, (60,), generator=g)] = 1e4
    near = 1.0 + eps * torch.randint(0, 9, (60, E), generator=g).float()
    low = torch.randn(60, E, generator=g)
    low[torch.rand(60, E, generator=g) < 0.8] = float("-inf")
    low[:, 0] = 0.25
    logits = [t.to(DT[dt]).to(DEV).requires_grad_() for t in (far, near, low)]
    r, _ = run(logits, K, 1.0, 0.0)
    assert torch.equal(r.expert_counts.cpu().long(), reference(logits, K, 1.0, 0.0)["counts"])


def test_inside_a_compiled_function():
    logits = draw(2, 60, 16, "fp32", 22)
    import pluggy_amd

    def f(a, b):
        return pluggy_amd.router_aux_loss([a * 2, b * 2], 16, 2, 1.0, 0.1).loss * 3

    want = f(*logits)
    got = torch.compile(f, backend="aot_eager")(*logits)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, logits), torch.autograd.grad(want, logits)):
        assert torch.equal(a, b)


def test_gradients_under_saved_tensor_hooks():
    """Hooks that give other tensors back (as activation offloading does), strided ones among them."""
    logits = draw(3, 40, 12, "fp32", 23)
    mask = torch.rand(40, generator=gen(23)) < 0.7
    r, want = run(logits, 3, 1.0, 0.5, mask.to(DEV))
    import pluggy_amd

    def unpack(t):
        t = t.clone()
        return t.t().contiguous().t() if t.dim() == 2 else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        r = pluggy_amd.router_aux_loss(logits, 12, 3, 1.0, 0.5, token_mask=mask.to(DEV))
    for a, b in zip(torch.autograd.grad(r.loss, logits), want):
        assert torch.equal(a, b)


def test_forward_in_a_graph():
    import pluggy_amd

    logits = [l.detach() for l in draw(3, 200, 32, "fp32", 19)]
    pluggy_amd.router_aux_loss(logits, 32, 4, 1.0, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        r = pluggy_amd.router_aux_loss(logits, 32, 4, 1.0, 1.0)
    for k in range(3):
        logits[1].mul_(1.1)
        graph.replay()
        want = pluggy_amd.router_aux_loss(logits, 32, 4, 1.0, 1.0)
        assert torch.equal(r.loss, want.loss) and torch.equal(r.expert_counts, want.expert_counts)
        torch.cuda.synchronize()


def test_backward_under_capture_raises():
    """Forward and backward recorded together: the node refuses before any launch, and eager work goes on."""
    import pluggy_amd

    logits = draw(1, 20, 8, "fp32", 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up, eagerly
        pluggy_amd.router_aux_loss(logits, 8, 2).loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want, logits[0].grad = logits[0].grad, None
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="not supported under HIP graph capture"):
        with torch.cuda.graph(graph):
            pluggy_amd.router_aux_loss(logits, 8, 2).loss.backward()
    torch.cuda.synchronize()
    logits[0].grad = None
    pluggy_amd.router_aux_loss(logits, 8, 2).loss.backward()
    assert torch.equal(logits[0].grad, want)


def test_host_tensors_from_a_hook_are_refused():
    """A hook that moves the saved logits to the host and forgets to bring them back."""
    import pluggy_amd

    logits = draw(2, 20, 8, "fp32", 24)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t if t.dim() == 2 else t.to(DEV)):
        r = pluggy_amd.router_aux_loss(logits, 8, 2)
    with pytest.raises(RuntimeError, match="ROCm GPU tensors only"):
        r.loss.backward()


@pytest.mark.parametrize("E,K", [(4, 1), (20, 3), (128, 4)])
def test_zeros_of_both_signs_at_the_top(E, K):
    """The largest logits are zeros of both signs, in either order, above others: equal, so the lower ids."""
    g = gen(25 + E)
    l = -1.0 - torch.rand(64, E, generator=g)
    for t in range(64):
        at = torch.randperm(E, generator=g)[:K + 1]
        l[t, at] = torch.where(torch.rand(K + 1, generator=g) < 0.5, 0.0, -0.0)
    logits = [l.to(DEV).requires_grad_()]
    r, grads = run(logits, K, 1.0, 0.1)
    ref = reference([torch.where(l == 0, 0.0, l)], K, 1.0, 0.1)
    check(r, grads, ref, 1.0, 0.1)


def test_some_layers_without_gradients():
    import pluggy_amd

    logits = draw(4, 30, 16, "fp32", 27)
    r, want = run(logits, 3, 1.0, 0.5)
    part = [l if i in (1, 3) else l.detach() for i, l in enumerate(logits)]
    r2 = pluggy_amd.router_aux_loss(part, 16, 3, 1.0, 0.5)
    got = torch.autograd.grad(r2.loss, [logits[1], logits[3]])
    assert torch.equal(r.loss, r2.loss) and torch.equal(got[0], want[1]) and torch.equal(got[1], want[3])
    assert not r2.load_balance.requires_grad and not r2.z_loss.requires_grad
    r3 = pluggy_amd.router_aux_loss([l.detach() for l in logits], 16, 3, 1.0, 0.5)
    assert torch.equal(r3.loss, r.loss) and not r3.loss.requires_grad
    with torch.no_grad():
        assert not pluggy_amd.router_aux_loss(logits, 16, 3).loss.requires_grad
    # the same layer twice: its gradients add up
    twice = pluggy_amd.router_aux_loss([logits[0], logits[0]], 16, 3, 1.0, 0.5)
    both = [logits[0].detach().clone().requires_grad_() for _ in range(2)]
    apart = torch.autograd.grad(pluggy_amd.router_aux_loss(both, 16, 3, 1.0, 0.5).loss, both)
    assert torch.equal(torch.autograd.grad(twice.loss, logits[0])[0], apart[0] + apart[1])


def test_backward_twice_and_with_a_kept_graph():
    import pluggy_amd

    logits = draw(2, 20, 8, "fp32", 28)
    loss = pluggy_amd.router_aux_loss(logits, 8, 2).loss
    first = torch.autograd.grad(loss, logits, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, logits), first))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, logits)
    loss = pluggy_amd.router_aux_loss(logits, 8, 2).loss
    with torch.no_grad():
        logits[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, logits)


def test_second_derivative_is_refused():
    import pluggy_amd

    logits = draw(2, 20, 8, "fp32", 29)
    got = torch.autograd.grad(pluggy_amd.router_aux_loss(logits, 8, 2).loss.square(), logits, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (got[0].sum() + got[1].sum()).backward()


def test_under_activation_checkpointing():
    from torch.utils.checkpoint import checkpoint

    import pluggy_amd

    logits = draw(3, 40, 16, "fp32", 30)

    def f(*ls):
        return pluggy_amd.router_aux_loss([l * 2 for l in ls], 16, 2, 1.0, 0.1).loss

    want = torch.autograd.grad(f(*logits), logits)
    got = torch.autograd.grad(checkpoint(f, *logits, use_reentrant=False), logits)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw

    import pluggy_amd

    l = torch.randn(20, 8, device=DEV)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            pluggy_amd.router_aux_loss([fw.make_dual(l, torch.ones_like(l))], 8, 2)


def test_past_32_bit_offsets():
    """2.2e9 logits: all rows counted, the last rows' gradients by the formula with the counts at hand."""
    import pluggy_amd

    N, E, K = 18000000, 128, 8
    l = torch.randn(N, E, device=DEV, dtype=torch.bfloat16).requires_grad_()
    r = pluggy_amd.router_aux_loss([l], E, K, 1.0, 1.0)
    (g,) = torch.autograd.grad(r.loss * N, [l])
    assert r.expert_counts.sum().item() == N * K
    f = r.expert_counts[0].double() / N - K / E
    for rows in (slice(0, 64), slice(N - 64, N)):
        p = torch.softmax(l[rows].detach().double(), -1)
        lse = torch.logsumexp(l[rows].detach().double(), -1)[:, None]
        m = (p * f).sum(-1, keepdim=True)
        want = p * (E * (f - m) + 2 * lse)
        bound = 96 * U * p * (E * (f.abs() + m.abs()) + 2 * (lse.abs() + 1))
        bound = bound + (want.abs() + bound) * torch.finfo(torch.bfloat16).eps / 2
        assert ((g[rows].double() - want).abs() <= bound + torch.finfo(torch.bfloat16).tiny).all()
