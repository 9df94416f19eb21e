"""gated_scan, gated_scan_step and rel_bias_attention under what watches autograd functions: forward-mode differentiation, which
they do not offer and must refuse, and torch.jit.trace, which must record the call and not the memory it writes.

On the CPU the library call is replaced by one that writes nothing: only the way to it is looked at."""
import pytest
import torch
from torch.autograd import forward_ad


def operators(dev, dtype=torch.float32):
    """(name, call, arguments) of every operator without gradients."""
    from unet_amd import ops
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(dev)
    x, gate, h0, table = r(2, 9, 16), r(2, 9, 16), r(2, 16).float(), r(8, 2).float()
    return [("gated_scan", lambda x, g, h0: ops.gated_scan(x, g, h0, return_state=True), (x, gate, h0)),
            ("rel_bias_attention", lambda q, k, v, t: ops.rel_bias_attention(q, k, v, t, 2, max_distance=5), (x, gate, r(2, 9, 16), table))]


@pytest.fixture
def hollow(monkeypatch):
    from unet_amd import ops
    monkeypatch.setattr(ops, "_run", lambda *a: None)
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)


def check_forward_mode(dev):
    from unet_amd import ops
    for name, call, args in operators(dev):
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                        call(*dual)
        with forward_ad.dual_level():               # a level without tangents of these inputs changes nothing
            call(*args)
    x, gate, state = (torch.zeros(2, 16, device=dev) for _ in range(3))
    for i in range(3):
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate((x, gate, state))]
            with pytest.raises(RuntimeError, match="tangents"):
                ops.gated_scan_step(*dual)
            ops.gated_scan_step(x, gate, state)


def check_traces(dev, compare):
    from unet_amd import ops
    for name, call, args in operators(dev):
        with torch.no_grad():
            traced = torch.jit.trace(call, args, check_trace=False)
            assert any(n.kind() == "prim::PythonOp" for n in traced.graph.nodes()), (name, traced.graph)
            if compare:
                fresh = [a * 0.5 + 0.25 for a in args]
                got, want = traced(*fresh), call(*fresh)
                for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                    assert torch.equal(a, b), name
    with torch.no_grad(), pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(ops.gated_scan_step, tuple(torch.zeros(2, 16, device=dev) for _ in range(3)), check_trace=False)


def test_forward_mode_is_refused_on_cpu(hollow):
    check_forward_mode("cpu")


def test_traces_hold_the_call_on_cpu(hollow):
    check_traces("cpu", False)


@pytest.mark.gpu
def test_forward_mode_is_refused():
    check_forward_mode("cuda")


@pytest.mark.gpu
def test_traces_hold_the_call():
    check_traces("cuda", True)
