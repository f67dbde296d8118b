"""GPU: layer norm forward and backward against the formulas in 64 bits.

Bounds, with u = 2^-24 and eps the output type's: a row's sums add at most
64 values in a thread and a tree over 256 threads (D = 64 + 8 steps), so the mean
is off by D u mean|x|, which counts relative to the deviation: k = (D + 16) u (1 +
|mu| / sd) relative to the terms of each result, plus half a step (eps / 2) of
the output type.
"""

from __future__ import annotations

import pytest
import torch

from tests._gpu_helpers import DEV, gen

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dt):
    return 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2


def tiny(dt):
    """Half of the smallest step near zero (subnormal results)."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def reference(x, w, b, eps, g, T, H):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    var = (x - mu).square().mean(-1, keepdim=True)
    sd = (var + eps).sqrt()
    xh = (x - mu) / sd
    w = torch.ones(H, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(H, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = xh * w + b
    k = 88 * U * (1 + mu.abs() / sd)
    out = {"y": (y, k * ((xh * w).abs() + w.abs() + b.abs()))}
    if g is not None:
        g = g.double()
        gw = g * w
        c1, c2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
        a1, a2 = gw.abs().mean(-1, keepdim=True), (gw * xh).abs().mean(-1, keepdim=True)
        out["gx"] = ((gw - c1 - xh * c2) / sd, 2 * k * (gw.abs() + a1 + (xh.abs() + 1) * a2 + a1) / sd)
        n = (T + 96) * U  # at most T additions, in pieces, and the joins
        out["gw"] = ((g * xh).sum(0), n * (g * xh).abs().sum(0) + (k * g.abs()).sum(0))
        out["gb"] = (g.sum(0), n * g.abs().sum(0))
    return out


def check(name, got, ref, bound):
    dt = got.dtype
    lim = bound + (ref.abs() + bound) * half_step(dt) + tiny(dt)
    err = (got.double() - ref).abs()
    worst = (err / lim).max().item() if err.numel() else 0.0
    print(f"{name}: worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0, f"{name}: {worst:.3f} times the bound"


def inputs(T, H, dt, wdt, seed, offset=0.3):
    g = gen(seed)
    x = (torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g)) + offset).to(DEV).to(dt)
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(DEV).to(wdt)
    b = (0.1 * torch.randn(H, generator=g)).to(DEV).to(wdt)
    return x, w, b, torch.randn(T, H, generator=g).to(DEV)


SIZES = [(1, 1), (1, 2048), (3, 8), (7, 511), (5, 513), (130, 1001), (64, 1024), (65, 2040), (33, 2056), (9, 4096),
         (7, 4104), (6, 8192), (5, 8200), (4, 16384), (3, 16385), (520, 17000), (4099, 96), (2500, 768)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("dt,out", [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "bf16"),
                                    ("fp32", "fp16")])
def test_forward_and_backward(T, H, dt, out):
    import pluggy_amd

    x, w, b, g = inputs(T, H, DT[dt], torch.float32, T * 31 + H)
    g = g.to(DT[out])
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = pluggy_amd.layer_norm(*leaves, 1e-5, DT[out])
    assert y.dtype == DT[out] and y.shape == x.shape
    with torch.no_grad():
        assert torch.equal(y, pluggy_amd.layer_norm(*leaves, 1e-5, DT[out]))
    gx, gw, gb = torch.autograd.grad(y, leaves, g)
    ref = reference(x, w, b, 1e-5, g, T, H)
    for name, got in (("y", y), ("gx", gx), ("gw", gw), ("gb", gb)):
        check(name, got.detach(), *ref[name])


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("wdt", ["fp32", "bf16", "fp16"])
def test_optional_and_typed_parameters(has_w, has_b, wdt):
    import pluggy_amd

    T, H = 70, 264
    x, w, b, g = inputs(T, H, torch.float32, DT[wdt], 5)
    leaves = [t.requires_grad_() for t in (x, w if has_w else None, b if has_b else None) if t is not None]
    y = pluggy_amd.layer_norm(x, w if has_w else None, b if has_b else None, 1e-6)
    grads = dict(zip(["gx"] + ["gw"] * has_w + ["gb"] * has_b, torch.autograd.grad(y, leaves, g)))
    ref = reference(x.detach(), w.detach() if has_w else None, b.detach() if has_b else None, 1e-6, g, T, H)
    check("y", y.detach(), *ref["y"])
    for name, got in grads.items():
        check(name, got, *ref[name])
        assert name == "gx" or got.dtype == DT[wdt]


def test_only_the_wanted_gradients_and_mixed_parameter_types():
    import pluggy_amd

    T, H = 40, 128
    x, w, b, g = inputs(T, H, torch.float32, torch.float32, 6)
    b16 = b.bfloat16().requires_grad_()
    y = pluggy_amd.layer_norm(x, w, b16)
    (gb,) = torch.autograd.grad(y, [b16], g)
    assert gb.dtype == torch.bfloat16
    check("gb", gb, *reference(x, w, b16.detach(), 1e-5, g, T, H)["gb"])


def test_large_mean_and_constant_rows():
    """A mean far above the deviation (the variance is not a difference of large sums), and rows without any."""
    import pluggy_amd

    x, w, b, g = inputs(20, 1024, torch.float32, torch.float32, 7, offset=1000.0)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = pluggy_amd.layer_norm(*leaves)
    ref = reference(x.detach(), w.detach(), b.detach(), 1e-5, g, 20, 1024)
    check("y", y.detach(), *ref["y"])
    check("gx", torch.autograd.grad(y, leaves, g)[0], *ref["gx"])
    flat = torch.full((3, 96), 7.0, device=DEV)
    assert torch.equal(pluggy_amd.layer_norm(flat), torch.zeros_like(flat))


def test_not_finite_rows_stay_apart():
    import pluggy_amd

    x, w, b, g = inputs(9, 256, torch.float32, torch.float32, 8)
    clean = pluggy_amd.layer_norm(x, w, b)
    x[4, 17] = float("inf")
    x[6, 0] = float("nan")
    y = pluggy_amd.layer_norm(x, w, b)
    for r in range(9):
        assert y[r].isnan().all() if r in (4, 6) else torch.equal(y[r], clean[r])


def test_shapes_strides_and_alignment():
    import pluggy_amd

    x, w, b, _ = inputs(24, 200, torch.bfloat16, torch.float32, 9)
    y = pluggy_amd.layer_norm(x, w, b)
    assert torch.equal(pluggy_amd.layer_norm(x.view(2, 3, 4, 200), w, b).view(24, 200), y)
    assert torch.equal(pluggy_amd.layer_norm(x.t().contiguous().t(), w, b), y)
    wide = torch.zeros(24, 333, dtype=torch.bfloat16, device=DEV)
    wide[:, 1:201] = x
    assert torch.equal(pluggy_amd.layer_norm(wide[:, 1:201], w, b), y)
    odd = torch.zeros(24 * 200 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(24, 200)  # starts on 2 bytes
    odd.copy_(x)
    ref = reference(x, w, b, 1e-5, None, 24, 200)
    check("odd", pluggy_amd.layer_norm(odd, w, b), *ref["y"])
    assert pluggy_amd.layer_norm(x[5], w, b).shape == (200,) and torch.equal(pluggy_amd.layer_norm(x[5], w, b), y[5])


@pytest.mark.parametrize("dt", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("H", [5, 127, 1000, 2047, 4095, 8191, 16383])
def test_rows_at_any_alignment(dt, H):
    """Rows, parameters and gradients that start on any element, and widths whose last chunk is cut."""
    import pluggy_amd

    T = 21
    x, w, b, g = inputs(T, H, DT[dt], torch.float32, H)
    g = g.to(DT[dt])

    def shifted(t, by):
        out = torch.zeros(t.numel() + by, dtype=t.dtype, device=DEV)[by:].view(t.shape)
        return out.copy_(t)

    leaves = [shifted(x, 3).requires_grad_(), shifted(w, 1).requires_grad_(), shifted(b, 2).requires_grad_()]
    y = pluggy_amd.layer_norm(*leaves)
    ref = reference(x, w, b, 1e-5, g, T, H)
    check("y", y.detach(), *ref["y"])
    for name, got in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, shifted(g, 1))):
        check(name, got, *ref[name])


@pytest.mark.parametrize("T,H", [(100003, 8), (70000, 40), (3000, 1024)])
def test_many_rows(T, H):
    """More rows than the grid has at a time."""
    import pluggy_amd

    x, w, b, g = inputs(T, H, torch.float32, torch.float32, H)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = pluggy_amd.layer_norm(*leaves)
    ref = reference(x.detach(), w.detach(), b.detach(), 1e-5, g, T, H)
    check("y", y.detach(), *ref["y"])
    for name, got in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, g)):
        check(name, got, *ref[name])


def test_no_rows():
    import pluggy_amd

    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    w, b = (torch.ones(64, device=DEV, requires_grad=True) for _ in range(2))
    y = pluggy_amd.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 64, device=DEV))
    assert gx.shape == (0, 64) and not gw.any() and not gb.any()


def test_gradient_matches_differences():
    """<grad, d> against the central difference of the 64-bit formula along d: the gradient's own error (the
    bounds above, summed over the direction) and the difference's, h^2 times the third derivative's scale."""
    import pluggy_amd

    T, H = 6, 48
    x, w, b, g = inputs(T, H, torch.float32, torch.float32, 10)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(pluggy_amd.layer_norm(*leaves), leaves, g)
    ds = [torch.randn(t.shape, generator=gen(11), dtype=torch.float64).to(DEV) for t in leaves]

    def loss(h):
        v = [t.detach().double() + h * d for t, d in zip(leaves, ds)]
        return (reference(*v, 1e-5, None, T, H)["y"][0] * g.double()).sum()

    h = 1e-4
    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((a.double() * d).sum() for a, d in zip(grads, ds))
    scale = sum((a.double().abs() * d.abs()).sum() for a, d in zip(grads, ds))
    assert abs(got - want) <= (400 * U + 100 * h * h) * scale


def test_deterministic_and_on_another_stream():
    import pluggy_amd

    x, w, b, g = inputs(3000, 768, torch.bfloat16, torch.float32, 12)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(pluggy_amd.layer_norm(*leaves), leaves, g.bfloat16())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = torch.autograd.grad(pluggy_amd.layer_norm(*leaves), leaves, g.bfloat16())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_forward_in_a_graph_and_backward_refused_there():
    import pluggy_amd

    x, w, b, _ = inputs(50, 512, torch.bfloat16, torch.float32, 13)
    with torch.no_grad():
        pluggy_amd.layer_norm(x, w, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pluggy_amd.layer_norm(x, w, b)
        for k in range(3):
            x.add_(0.5)
            graph.replay()
            assert torch.equal(y, pluggy_amd.layer_norm(x, w, b))
            torch.cuda.synchronize()


def test_backward_under_capture_raises():
    """Forward and backward recorded together: the node refuses before any launch, and eager work goes on."""
    import pluggy_amd

    x, w, b, _ = inputs(8, 64, torch.float32, torch.float32, 14)
    x.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up, eagerly
        pluggy_amd.layer_norm(x, w, b).sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want, x.grad = x.grad, None
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="not supported under HIP graph capture"):
        with torch.cuda.graph(graph):
            pluggy_amd.layer_norm(x, w, b).sum().backward()
    torch.cuda.synchronize()
    x.grad = None
    pluggy_amd.layer_norm(x, w, b).sum().backward()
    assert torch.equal(x.grad, want)


def test_second_derivative_is_refused():
    import pluggy_amd

    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    (gx,) = torch.autograd.grad(pluggy_amd.layer_norm(x).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


def test_compiled_matches_eager():
    import pluggy_amd

    x, w, b, g = inputs(33, 256, torch.float32, torch.float32, 15)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def f(x, w, b):
        return pluggy_amd.layer_norm(x, w, b, 1e-5, torch.bfloat16) * 2

    y = f(*leaves)
    yc = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(y, yc)
    grads = torch.autograd.grad(y, leaves, g.bfloat16()), torch.autograd.grad(yc, leaves, g.bfloat16())
    assert all(torch.equal(a, c) for a, c in zip(*grads))


@pytest.mark.parametrize("amp", [False, True])
def test_moe_sublayer_with_a_layer_norm(amp):
    """``moe_sublayer`` runs a LayerNorm block: x + mlp(layer_norm(x)) with the same calls."""
    import pluggy_amd

    B, S, H = 2, 19, 64
    torch.manual_seed(0)
    mlp = pluggy_amd.Qwen3MoeSparseMLP(H, 32, 8, 2).to(DEV)
    for p in mlp.parameters():
        torch.nn.init.normal_(p, std=0.1)
    norm = torch.nn.LayerNorm(H).to(DEV)
    torch.nn.init.normal_(norm.weight, mean=1.0, std=0.1)
    x = torch.randn(B, S, H, device=DEV, requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16, enabled=amp):
        y = pluggy_amd.moe_sublayer(x, norm, mlp)
        normed = pluggy_amd.layer_norm(x, norm.weight, norm.bias, norm.eps, torch.bfloat16 if amp else None)
        want = x + mlp(normed)
    assert y.dtype == torch.float32 and torch.equal(y, want)
    params = [x, norm.weight, norm.bias, *mlp.parameters()]
    g = torch.randn_like(y)
    for a, c in zip(torch.autograd.grad(y, params, g), torch.autograd.grad(want, params, g)):
        assert torch.equal(a, c) and a.abs().sum() > 0


def test_host_tensors_from_a_hook_are_refused():
    import pluggy_amd

    x, w, b, g = inputs(8, 64, torch.float32, torch.float32, 26)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        y = pluggy_amd.layer_norm(x.requires_grad_(), w, b)
    with pytest.raises(RuntimeError, match="ROCm GPU tensors only"):
        torch.autograd.grad(y, [x], g)


@pytest.mark.parametrize("which", ["x", "w", "b", "xb", "wb", "no w", "no b"])
def test_gradients_of_any_subset(which):
    """A gradient does not depend on which others are asked for."""
    import pluggy_amd

    x, w, b, g = inputs(40, 96, torch.float32, torch.float32, 27)
    if which == "no w":
        w = None
    if which == "no b":
        b = None
    given = {"x": x, "w": w, "b": b}
    full = {k: t.clone().requires_grad_() for k, t in given.items() if t is not None}
    y = pluggy_amd.layer_norm(full["x"], full.get("w"), full.get("b"))
    want = dict(zip(full, torch.autograd.grad(y, list(full.values()), g)))
    names = [k for k in "xwb" if k in which] if not which.startswith("no") else ["x", "wb".replace(which[-1], "")]
    leaves = {k: given[k].clone().requires_grad_() for k in names}
    args = {k: leaves.get(k, t) for k, t in given.items()}
    y = pluggy_amd.layer_norm(args["x"], args["w"], args["b"])
    for k, got in zip(names, torch.autograd.grad(y, list(leaves.values()), g)):
        assert torch.equal(got, want[k])


def test_backward_twice_and_with_a_kept_graph():
    import pluggy_amd

    x, w, b, g = inputs(8, 64, torch.float32, torch.float32, 28)
    y = pluggy_amd.layer_norm(x.requires_grad_(), w, b)
    first = torch.autograd.grad(y, [x], g, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, [x], g)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, [x], g)
    y = pluggy_amd.layer_norm(x, w, b)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], g)


@pytest.mark.parametrize("reentrant", [False, True])
def test_under_activation_checkpointing(reentrant):
    """Computed again in the backward, where the second forward stops as soon as what is needed is there."""
    from torch.utils.checkpoint import checkpoint

    import pluggy_amd

    x, w, b, g = inputs(40, 96, torch.float32, torch.float32, 29)
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def f(x, w, b):
        return pluggy_amd.layer_norm(x * 2, w, b).sin()

    want = torch.autograd.grad(f(*leaves), leaves, g)
    if reentrant:
        checkpoint(f, *leaves, use_reentrant=True).backward(g)
        got = [t.grad for t in leaves]
    else:
        got = torch.autograd.grad(checkpoint(f, *leaves, use_reentrant=False), leaves, g)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw

    import pluggy_amd

    x = torch.randn(4, 64, device=DEV)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            pluggy_amd.layer_norm(fw.make_dual(x, torch.ones_like(x)))


def test_without_gradients_the_same_values():
    import pluggy_amd

    x, w, b, _ = inputs(33, 257, torch.float32, torch.float32, 30)
    want = pluggy_amd.layer_norm(x.clone().requires_grad_(), w, b).detach()
    assert torch.equal(pluggy_amd.layer_norm(x, w, b), want)
    with torch.no_grad():
        y = pluggy_amd.layer_norm(x.requires_grad_(), w, b)
    assert torch.equal(y, want) and not y.requires_grad
    with torch.inference_mode():
        assert torch.equal(pluggy_amd.layer_norm(x.detach(), w, b), want)


@pytest.mark.parametrize("H", [2001, 17000])
def test_past_32_bit_offsets(H):
    """2.2e9 values, held in registers and walked in passes: the last rows are those of the rows by themselves."""
    import pluggy_amd

    T = 2200000000 // H
    x = torch.randn(T, H, device=DEV, dtype=torch.bfloat16).requires_grad_()
    w, b = torch.rand(H, device=DEV) + 0.5, torch.randn(H, device=DEV)
    g = torch.randn(T, H, device=DEV, dtype=torch.bfloat16)
    y = pluggy_amd.layer_norm(x, w, b)
    gx = torch.autograd.grad(y, [x], g)[0]
    for rows in (slice(0, 40), slice(T - 40, T)):
        part = x[rows].detach().requires_grad_()
        yp = pluggy_amd.layer_norm(part, w, b)
        assert torch.equal(y[rows], yp)
        assert torch.equal(gx[rows], torch.autograd.grad(yp, [part], g[rows])[0])


def test_from_several_threads_on_their_own_streams():
    """Calls at once: each thread's results are those of the same work alone."""
    import threading

    import pluggy_amd

    def work(k):
        x, w, b, g = inputs(200 + k, 333, torch.float32, torch.float32, 40 + k)
        leaves = [t.requires_grad_() for t in (x, w, b)]
        logits = [torch.randn(100 + k, 24, generator=gen(50 + k)).to(DEV).requires_grad_() for _ in range(3)]
        out = []
        for _ in range(10):
            y = pluggy_amd.layer_norm(*leaves)
            r = pluggy_amd.router_aux_loss(logits, 24, 3, 1.0, 0.1)
            out.append([y, r.loss, *torch.autograd.grad(y, leaves, g), *torch.autograd.grad(r.loss, logits)])
        return out

    alone = [work(k) for k in range(4)]
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got[k] = work(k)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k in range(4):
        assert all(torch.equal(a, b) for u, v in zip(got[k], alone[k]) for a, b in zip(u, v))
