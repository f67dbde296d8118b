"""Refusals of the training operators (auxiliary loss, layer norm, 8-bit checkpoints): bad arguments are
turned down on the host, before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from pluggy_amd import _lib

    return _lib.load()


FAKE = ctypes.c_void_p(256)  # never read: every call here is refused first


def message(lib):
    return lib.pmoe_last_error_string().decode()


def rows(*n):
    return (ctypes.c_int64 * len(n))(*n)


def pointers(n, value=256):
    return (ctypes.c_void_p * n)(*[value] * n)


def aux(lib, logits=None, counts=None, L=2, dtype=0, mask=None, mask_rows=0, E=8, K=2, ws=FAKE, nbytes=1 << 20,
        out=FAKE):
    return lib.pmoe_aux_loss_forward(logits if logits is not None else pointers(2),
                                     counts if counts is not None else rows(5, 5), L, dtype, mask, mask_rows, E, K,
                                     1.0, 1.0, out, FAKE, FAKE, FAKE, FAKE, ws, nbytes, None)


@pytest.mark.parametrize("kw,code,needle", [
    ({"L": 0}, -1, "layers"),
    ({"L": 5000}, -1, "layers"),
    ({"K": 9}, -1, "exceeds num_experts"),
    ({"E": 2000}, -1, "> 1024"),
    ({"K": 0}, -1, "positive"),
    ({"E": 100, "K": 65}, -1, "> 64"),
    ({"dtype": 7}, -1, "dtype"),
    ({"dtype": 3}, -1, "dtype"),
    ({"counts": rows(5, -1)}, -1, "rows"),
    ({"counts": rows(1 << 30, 1 << 30)}, -1, "rows in all"),
    ({"logits": pointers(2, 0)}, -1, "null tensor"),
    ({"out": None}, -1, "null tensor"),
    ({"mask": FAKE, "mask_rows": 4}, -1, "a mask of 4 rows"),
    ({"nbytes": 64}, -3, "workspace"),
    ({"ws": None}, -3, "workspace"),
])
def test_aux_loss_refusals(lib, kw, code, needle):
    assert aux(lib, **kw) == code and needle in message(lib)


def test_aux_loss_backward_and_statistics_refusals(lib):
    rc = lib.pmoe_aux_loss_backward(pointers(2), pointers(2), rows(5, 6), 2, 0, FAKE, 5, 8, FAKE, FAKE, 1.0, 1.0, None)
    assert rc == -1 and "a mask of 5 rows, but layer 1 has 6" in message(lib)
    rc = lib.pmoe_aux_loss_backward(pointers(2), pointers(2), rows(5, 6), 2, 0, None, 0, 8, None, FAKE, 1.0, 1.0, None)
    assert rc == -1 and "null tensor" in message(lib)
    # nothing to write: no rows
    assert lib.pmoe_aux_loss_backward(pointers(2, 0), pointers(2, 0), rows(0, 0), 2, 0, None, 0, 8, FAKE, FAKE, 1.0,
                                      1.0, None) == 0

    def stats(L=2, n=10, E=8, K=2, p=None, nbytes=1 << 20):
        p = p if p is not None else pointers(2)
        return lib.pmoe_aux_loss_from_stats(p, pointers(2), pointers(2), L, n, E, K, 1.0, 1.0, FAKE, FAKE, FAKE, FAKE,
                                            FAKE, FAKE, nbytes, None)

    assert stats(L=0) == -1 and stats(n=-1) == -1 and stats(K=9) == -1
    assert stats(p=pointers(2, 0)) == -1 and "null tensor" in message(lib)
    assert stats(nbytes=8) == -3


def norm_fwd(lib, T=4, H=8, x=0, w=0, y=0, eps=1e-5, px=FAKE, mean=None, rstd=None):
    return lib.pmoe_layernorm_forward(px, x, None, None, w, eps, T, H, FAKE, y, mean, rstd, None)


@pytest.mark.parametrize("kw,code,needle", [
    ({"T": -1}, -1, "sizes"),
    ({"H": 0}, -1, "sizes"),
    ({"H": 1 << 31}, -1, "sizes"),
    ({"T": 1 << 31}, -1, "sizes"),
    ({"T": 1 << 23, "H": 16385}, -2, "one launch"),
    ({"x": 1, "y": 0}, -1, "x's type"),
    ({"x": 1, "y": 2}, -1, "x's type"),
    ({"x": 5}, -1, "dtype"),
    ({"w": -1}, -1, "dtype"),
    ({"eps": -1.0}, -1, "eps"),
    ({"eps": float("nan")}, -1, "eps"),
    ({"mean": FAKE}, -1, "together"),
    ({"px": None}, -1, "null tensor"),
])
def test_layernorm_forward_refusals(lib, kw, code, needle):
    assert norm_fwd(lib, **kw) == code and needle in message(lib)


def test_layernorm_backward_refusals(lib):
    def bwd(T=4, H=8, g=0, x=0, mean=FAKE, ws=FAKE, nbytes=1 << 20):
        return lib.pmoe_layernorm_backward(FAKE, g, FAKE, x, None, 0, mean, FAKE, T, H, FAKE, FAKE, FAKE, ws, nbytes,
                                           None)

    assert bwd(g=0, x=1) == -1 and bwd(T=1 << 23, H=20000) == -2
    assert lib.pmoe_layernorm_backward_workspace_size(0, 8) == 0
    assert lib.pmoe_layernorm_backward_workspace_size(1000, 2048) >= 2 * 125 * 2048 * 4
    assert bwd(mean=None) == -1 and "null tensor" in message(lib)
    assert bwd(nbytes=0) == -3 and bwd(ws=None) == -3
    assert bwd(ws=ctypes.c_void_p(260)) == -1 and "aligned" in message(lib)


def test_act8_refusals(lib):
    assert lib.pmoe_act8_save(FAKE, 0, -1, 8, FAKE, FAKE, None) == -1
    assert lib.pmoe_act8_save(FAKE, 0, 4, 0, FAKE, FAKE, None) == -1
    assert lib.pmoe_act8_save(FAKE, 4, 4, 8, FAKE, FAKE, None) == -1 and "dtype" in message(lib)
    assert lib.pmoe_act8_save(None, 0, 4, 8, FAKE, FAKE, None) == -1 and "null" in message(lib)
    assert lib.pmoe_act8_save(FAKE, 0, 1 << 31, 32, FAKE, FAKE, None) == -2 and "one launch" in message(lib)
    assert lib.pmoe_act8_restore(None, FAKE, 4, 8, FAKE, 0, None) == -1
    assert lib.pmoe_act8_restore(FAKE, FAKE, 1 << 40, 8, FAKE, 0, None) == -2
    assert lib.pmoe_act8_save(FAKE, 0, 0, 8, None, None, None) == 0  # no rows: nothing to do

    def gate_up(P=4, H=8, I=8, dtype=1, codes=FAKE, ws=FAKE, nbytes=1 << 20):
        return lib.pmoe_gate_up_swiglu_act8(FAKE, None, None, P, FAKE, FAKE, dtype, P, 2, H, I, codes, FAKE, FAKE, ws,
                                            nbytes, None)

    assert gate_up(I=12) == -1 and "multiple of 8" in message(lib)
    assert gate_up(I=0) == -1 and gate_up(dtype=3) == -1 and gate_up(codes=None) == -1
    need = lib.pmoe_gate_up_swiglu_act8_workspace_size(4, 2, 8, 8, 1)
    if need:
        assert gate_up(nbytes=need - 1) == -3

    def dgrad(P=4, H=8, I=8, dtype=1, part=None, ld=0, weight=FAKE, nbytes=1 << 20):
        return lib.pmoe_down_proj_dgrad_act8(FAKE, None, weight, P, FAKE, FAKE, FAKE, FAKE, dtype, P, 2, H, I, None,
                                             FAKE, part, ld, FAKE, nbytes, None)

    assert dgrad() == -1 and "null tensor" in message(lib)
    assert dgrad(H=12) == -1 and dgrad(dtype=9) == -1


def test_python_refusals():
    """Shapes, types and devices, before the library is asked."""
    import pluggy_amd
    from pluggy_amd import ops

    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pluggy_amd.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.act8_save(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.act8_restore(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pluggy_amd.router_aux_loss([x], 8, 2)
    with pytest.raises(AssertionError):
        pluggy_amd.layer_norm(x, torch.ones(7))
    with pytest.raises(AssertionError):
        pluggy_amd.layer_norm(torch.tensor(1.0))
    with pytest.raises(AssertionError):
        pluggy_amd.router_aux_loss([x], 9, 2)
    with pytest.raises(AssertionError):
        pluggy_amd.router_aux_loss([x], 8, 9)
    with pytest.raises(AssertionError):
        pluggy_amd.router_aux_loss([x, x.half()], 8, 2)
    empty = pluggy_amd.router_aux_loss([], 8, 2)
    assert empty.loss.item() == 0.0 and empty.expert_counts.shape == (0, 8)


def test_fake_shapes_of_the_checkpointed_ops():
    """The ops' shape functions with an 8-bit checkpoint: codes and exps in place of the two saved tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    import pluggy_amd  # noqa: F401 - registers the ops

    with FakeTensorMode():
        T, K, E, H, I = 6, 2, 4, 64, 40
        hid = torch.empty(T, H, dtype=torch.bfloat16)
        idx, w = torch.empty(T, K, dtype=torch.int64), torch.empty(T, K)
        gu, dn = torch.empty(E, 2 * I, H, dtype=torch.bfloat16), torch.empty(E, H, I, dtype=torch.bfloat16)
        out = torch.ops.pmoe.expert_ffn_fwd(hid, idx, w, gu, dn, None, None, True)
        assert out[5].shape == (T * K, 2 * I) and out[5].dtype == torch.int8
        assert out[6].shape == (T * K, 2, 2) and out[6].dtype == torch.uint8
        plain = torch.ops.pmoe.expert_ffn_fwd(hid, idx, w, gu, dn)
        assert plain[5].dtype == torch.bfloat16 and plain[6].shape == (T * K, I)
        y, stats = torch.ops.pmoe.layer_norm_fwd(torch.empty(3, 5, 8), None, None, 1e-5, torch.float16)
        assert y.shape == (3, 5, 8) and y.dtype == torch.float16 and stats.shape == (2, 15)


def test_the_autograd_nodes_load_over_the_same_library(lib):
    """The nodes link against the library that is loaded; one that is missing is named in the error."""
    from pluggy_amd import _lib

    assert {"layer_norm", "aux_loss"} <= set(dir(_lib.nodes()))
    mapped = {line.split()[-1] for line in open("/proc/self/maps") if line.rstrip().endswith("libpmoe.so")}
    assert len(mapped) == 1
    assert lib.pmoe_stream_capturing(None) == 0


def test_missing_autograd_nodes_are_an_error(monkeypatch):
    import sys

    from pluggy_amd import _lib

    monkeypatch.setattr(_lib, "_nodes", None)
    monkeypatch.setitem(sys.modules, "pluggy_amd._autograd", None)
    monkeypatch.delattr("pluggy_amd._autograd", raising=False)
    with pytest.raises(RuntimeError, match="python -m pluggy_amd.build"):
        _lib.nodes()
