"""The autograd nodes of qk_norm_rope and linear_attn_func: the native ones and the
Python Functions that stand in for them behave alike."""
import pytest
import torch

import tilelang_fa_v100 as fa
from helpers import randn
from tilelang_fa_v100 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rope_call(seed=0, kind="both"):
    g = torch.Generator().manual_seed(seed)
    q, k = (randn(g, 2, 33, h, 64, dtype=torch.bfloat16).to(DEV).requires_grad_() for h in (4, 2))
    w = [(1 + 0.1 * torch.randn(64, generator=g)).to(DEV).requires_grad_() for _ in range(2)]
    cos, sin = (torch.randn(33, 32, generator=g).to(DEV) for _ in range(2))
    qw, kw = (w[0], w[1]) if kind == "both" else (w[0], None) if kind == "q" else (None, None)
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    return lambda: fa.qk_norm_rope(q, k, cos, sin, qw, kw), leaves, q


def linear_call(seed=0, kind="state"):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (randn(g, 1, 70, h, 64, dtype=torch.float16).to(DEV).requires_grad_()
               for h in (4, 2, 2))
    s = torch.randn(1, 4, 64, 64, generator=g).to(DEV).requires_grad_()
    decay = -torch.rand(4, generator=g).to(DEV)
    if kind == "state":
        return (lambda: fa.linear_attn_func(q, k, v, decay, initial_state=s,
                                            return_final_state=True)), [q, k, v, s], k
    return (lambda: (fa.linear_attn_func(q, k, v, decay),)), [q, k, v], k


CALLS = {"rope": rope_call, "rope_q": lambda: rope_call(1, "q"), "turn": lambda: rope_call(2, ""),
         "linear_state": linear_call, "linear": lambda: linear_call(1, "")}


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_native, "_missing", True)
    return request.param


@pytest.mark.parametrize("name", CALLS)
def test_native_and_python_gradients_are_the_same_bits(name, monkeypatch):
    call, leaves, _ = CALLS[name]()
    out = call()
    assert "Backward" in type(out[0].grad_fn).__name__ or "Backward" in out[0].grad_fn.name()
    g = [torch.randn_like(o) for o in out]
    native = torch.autograd.grad(out, leaves, g)
    monkeypatch.setattr(_native, "_missing", True)
    out2 = call()
    python = torch.autograd.grad(out2, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip((*out, *native), (*out2, *python)))


@pytest.mark.parametrize("name", CALLS)
def test_partial_and_odd_gradients(name, path):
    """One output's gradient alone, expanded or misaligned; some of the leaves."""
    call, leaves, _ = CALLS[name]()
    out = call()
    want = torch.autograd.grad(out, leaves, [torch.ones_like(out[0])]
                               + [torch.zeros_like(o) for o in out[1:]])
    out = call()
    got = torch.autograd.grad(out[0], leaves, torch.ones((), dtype=out[0].dtype, device=DEV)
                              .expand_as(out[0]))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    out = call()
    got = torch.autograd.grad(out[0].sum(), leaves[1])
    assert torch.equal(got[0], want[1])
    out = call()
    odd = torch.ones(out[0].numel() + 1, dtype=out[0].dtype, device=DEV)[1:].view_as(out[0])
    got = torch.autograd.grad(out[0], leaves, odd)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", CALLS)
def test_graph_rules(name, path):
    """A second backward needs retain_graph, a second derivative is an error, and an
    input changed in place is noticed (where the backward reads it)."""
    call, leaves, saved = CALLS[name]()
    out = call()
    loss = sum(o.float().sum() for o in out)
    loss.backward(retain_graph=True)
    first = [t.grad.clone() for t in leaves]
    loss.backward()
    assert all(torch.equal(2 * a, t.grad) for a, t in zip(first, leaves))
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    out = call()
    g = torch.ones_like(out[0]).requires_grad_()
    grads = torch.autograd.grad(out[0], leaves[0], g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        torch.autograd.grad(grads[0].float().sum(), g)
    if name != "turn":
        out = call()
        with torch.no_grad():
            saved.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out[0].float().sum().backward()


@pytest.mark.parametrize("name", CALLS)
def test_backward_on_a_side_stream_and_in_a_graph(name, path):
    call, leaves, _ = CALLS[name]()

    def step():
        out = call()
        return torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        with torch.no_grad():
            leaves[0].mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(step(), kept))


@pytest.mark.parametrize("name", CALLS)
def test_a_capture_beside_a_live_eager_graph_is_refused(name):
    """A graph of the same leaves made before the capture lives: the call refuses (the
    engine would end the process at the captured backward).  Without it, or on
    detached leaves, the step is captured."""
    call, leaves, _ = CALLS[name]()
    live = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="live autograd graph"):
        with torch.cuda.graph(graph):
            call()
    del live
    want = call()
    want = [t.clone() for t in torch.autograd.grad(want, leaves, [torch.ones_like(o) for o in want])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
        grads = torch.autograd.grad(out, leaves, [torch.ones_like(o) for o in out])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, grads))
