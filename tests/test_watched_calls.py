"""Calls without gradients go to the library directly; those that a trace, a function transform or forward-mode
differentiation watches must not: the watcher sees the operator's Function, or the call is refused. (On the CPU, with a
stand-in for the launch.)"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import trident_b200 as trident
from trident_b200 import _lib

F = trident.function


@pytest.fixture
def calls(monkeypatch):
    """Stand-ins that fill outputs with ones; the list of entry points that were called."""
    seen = []

    def stand_in(name, outputs):
        def run(*args):
            seen.append(name)
            for t in filter(torch.is_tensor, args[:outputs]):
                with torch.inference_mode(t.is_inference()):
                    t.data.fill_(1.0)  # (as a kernel: autograd sees nothing of it)

        monkeypatch.setattr(_lib, name, run)

    monkeypatch.setattr(_lib, "require_one_device", lambda *tensors: None)
    monkeypatch.setattr(_lib, "paged_attention_workspace", lambda *args: 0)
    stand_in("window_attention_fwd", 1)
    stand_in("gated_residual_rms_norm_fwd", 2)
    for name in ("window_attention_bwd_workspace", "gated_residual_rms_norm_bwd_workspace"):
        monkeypatch.setattr(_lib, name, lambda *args: 16)
    stand_in("window_attention_bwd", 3)
    stand_in("gated_residual_rms_norm_bwd", 5)
    stand_in("paged_attention", 1)
    stand_in("paged_cache_append", 0)
    return seen


def _window(q):
    return F.sliding_window_attention(q, q, q, 4)


def _norm(x):
    return F.gated_residual_rms_norm(x, x, None, torch.ones(16))[0]


Q = torch.randn(1, 2, 8, 16)
TABLE, LENGTHS, POOL = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.zeros(4, 8, 2, 16)


def _paged(q):
    return F.paged_attention(q, POOL, POOL, TABLE, LENGTHS)


def _append(k):
    return F.paged_cache_append(k, k, POOL, POOL, TABLE, LENGTHS)


@pytest.mark.parametrize("call", [_window, _norm])
def test_forward_mode_is_refused(call, calls):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            call(forward_ad.make_dual(Q, torch.ones_like(Q)))
        assert torch.all(call(Q) == 1)  # nothing to differentiate
    with torch.no_grad(), forward_ad.dual_level(), pytest.raises(NotImplementedError, match="jvp"):
        call(forward_ad.make_dual(Q, torch.ones_like(Q)))


@pytest.mark.parametrize("call", [_window, _norm])
def test_transforms_are_refused(call, calls):
    for run in (lambda: torch.func.jvp(call, (Q,), (Q,)), lambda: torch.func.vmap(call)(Q[None])):
        with pytest.raises(RuntimeError, match="setup_context"):
            run()


@pytest.mark.parametrize("call, name", [(_window, "WindowAttention"), (_norm, "GatedResidualRMSNorm")])
@pytest.mark.filterwarnings("ignore")
def test_a_trace_records_the_function(call, name, calls):
    traced = torch.jit.trace(call, (Q,), check_trace=False)
    graph = traced.graph
    nodes = [n.kind() for n in graph.nodes()]
    assert "prim::PythonOp" in nodes and "aten::empty_like" not in nodes, graph
    assert name in str(graph)
    before = len(calls)
    assert torch.all(traced(Q) == 1) and len(calls) == before + 1


@pytest.mark.parametrize("call", [_paged, _append])
@pytest.mark.filterwarnings("ignore")
def test_paged_calls_are_refused(call, calls):
    x = torch.randn(3, 2, 16)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        call(x)
    assert len(calls) == 1
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    for run in (lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.vmap(call)(x[None])):
        with pytest.raises(ValueError, match="transforms"):
            run()
    assert len(calls) == 1


def test_ordinary_calls_are_direct(calls):
    for call, name in ((_window, "window_attention_fwd"), (_norm, "gated_residual_rms_norm_fwd")):
        assert call(Q).grad_fn is None and calls[-1] == name
        assert call(Q.clone().requires_grad_(True)).grad_fn is not None


@pytest.mark.parametrize("which", ["key_cache", "value_cache", "a view", "output"])
def test_autograd_sees_what_is_written(which, calls):
    """A graph that saved a tensor which a call writes in place refuses its backward pass."""
    keys, values, out, x = torch.randn(4, 8, 2, 16), torch.randn(4, 8, 2, 16), torch.randn(3, 2, 16), torch.randn(3, 2, 16)
    saved = {"key_cache": keys, "value_cache": values, "a view": keys[1], "output": out}[which]
    leaf = torch.randn_like(saved, requires_grad=True)
    loss = (saved * leaf).sum()
    F.paged_attention(x, keys, values, TABLE, LENGTHS)  # reads
    torch.autograd.grad(loss, leaf, retain_graph=True)
    if which == "output":
        F.paged_attention(x, keys, values, TABLE, LENGTHS, output=out)
    else:
        F.paged_cache_append(x, x, keys, values, TABLE, LENGTHS)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_are_written(calls):
    with torch.inference_mode():
        keys, x = torch.zeros(4, 8, 2, 16), torch.zeros(3, 2, 16)
        out = F.paged_attention(x, keys, keys, TABLE, LENGTHS, output=x)
    with torch.no_grad():
        F.paged_cache_append(x, x, keys, keys, TABLE, LENGTHS)
        assert F.paged_attention(x, keys, keys, TABLE, LENGTHS, output=out) is out
    assert len(calls) == 3


@pytest.mark.parametrize("call", [_window, _norm])
def test_a_second_derivative_is_refused(call, calls):
    """Its part of a sum is not dropped without a word, whether or not the gradient that comes in needs one itself."""
    for ask in (False, True):
        x = Q.clone().requires_grad_(True)
        out = call(x)
        dout = torch.ones_like(out, requires_grad=ask)
        (dx,) = torch.autograd.grad(out, x, dout, create_graph=True)
        assert dx.requires_grad
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(dx.square().sum() + x.square().sum(), x)
    x = Q.clone().requires_grad_(True)
    call(x).sum().backward()
    assert not x.grad.requires_grad
