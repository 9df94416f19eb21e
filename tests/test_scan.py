"""The gated linear recurrence (ops.gated_scan, ops.gated_scan_step): refusals on the CPU, values and gradients on the GPU
against a row-by-row evaluation in float64.

Tolerances come from a running error bound evaluated next to the float64 recurrence.  With u = 2^-24 the kernel's gate has a
relative error of at most K u: its exponential's argument is rounded twice (2 |g| u for |g| <= 10), exponential, sum, reciprocal
and product add up to 6 units, and a product of gates adds one rounding a row.  K = 40 covers |g| <= 10 with room for the one
rounding of each fused step.  So the state's error obeys e_t <= f_t e_{t-1} + K u (f_t |h_{t-1}| + (1 - f_t) |x_t|), the
adjoint's the same recurrence from the other end, and a bf16 result is half a step, 2^-8 relative, further off."""
import ctypes as C

import pytest
import torch

U, K = 2.0 ** -24, 40.0


def oracle(x, g, h0, dh, dlast, reverse):
    """float64 values and error bounds: h, last, dx, dg, dh0 and the bound of each."""
    x, g = x.double().cpu(), g.double().cpu()
    if reverse:
        x, g = x.flip(1), g.flip(1)
    n, l, c = x.shape
    f, keep = torch.sigmoid(g), torch.sigmoid(-g)
    s = torch.zeros(n, c, dtype=torch.float64) if h0 is None else h0.double().cpu()
    e = torch.zeros_like(s)
    h, eh, before, eb = (torch.empty_like(x) for _ in range(4))
    for t in range(l):
        before[:, t], eb[:, t] = s, e
        e = f[:, t] * e + K * U * (f[:, t] * s.abs() + keep[:, t] * x[:, t].abs())
        s = f[:, t] * s + keep[:, t] * x[:, t]
        h[:, t], eh[:, t] = s, e
    out = dict(h=(h, eh), last=(s, e))
    if dh is not None:
        d = dh.double().cpu()
        d = d.flip(1) if reverse else d
        mu = torch.zeros_like(s) if dlast is None else dlast.double().cpu()
        em = torch.zeros_like(s)
        dx, dg, ex, eg = (torch.empty_like(x) for _ in range(4))
        for t in range(l - 1, -1, -1):
            lam, el = d[:, t] + mu, em + U * (d[:, t].abs() + mu.abs())
            diff, ed = before[:, t] - x[:, t], eb[:, t] + U * (before[:, t].abs() + x[:, t].abs())
            fk = f[:, t] * keep[:, t]
            dx[:, t], ex[:, t] = keep[:, t] * lam, keep[:, t] * (el + 2 * K * U * lam.abs())
            dg[:, t] = lam * diff * fk
            eg[:, t] = fk * (el * diff.abs() + lam.abs() * ed + 3 * K * U * (lam * diff).abs())
            mu, em = f[:, t] * lam, f[:, t] * (el + K * U * lam.abs())
        out.update(dx=(dx, ex), dg=(dg, eg), dh0=(mu, em))
    if reverse:
        for k in ("h", "dx", "dg"):
            if k in out:
                out[k] = tuple(v.flip(1) for v in out[k])
    return out


def near(got, want, what=""):
    value, bound = want
    half = torch.finfo(got.dtype).eps / 2
    got = got.detach().double().cpu()
    tol = bound * (1 + half) + half * value.abs() + 1e-37
    bad = (got - value).abs() > tol
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - value).abs() / tol).max()):.2f} tolerances"
    assert bool(torch.isfinite(got).all())


def inputs(n, l, c, dtype, seed=0, dev="cuda", spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    gate = (r(n, l, c) + spread * r(1, 1, c)).clamp(-10, 10)
    return (r(n, l, c).to(dtype).to(dev), gate.to(dtype).to(dev), r(n, c).to(dev), r(n, l, c).to(dtype).to(dev), r(n, c).to(dev))


def call(x, g, h0, dh, dlast, reverse):
    from unet_amd import ops
    x, g = x.detach().requires_grad_(), g.detach().requires_grad_()
    h0 = None if h0 is None else h0.detach().requires_grad_()
    h, last = ops.gated_scan(x, g, h0, reverse=reverse, return_state=True)
    outs, grads = [h], [dh]
    if dlast is not None:
        outs.append(last)
        grads.append(dlast)
    leaves = [x, g] + ([] if h0 is None else [h0])
    got = torch.autograd.grad(outs, leaves, grads)
    return dict(zip(("h", "last", "dx", "dg", "dh0"), (h, last) + got))


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_gradients_against_autograd_on_cpu():
    x, g, h0, dh, dlast = (t.double() for t in inputs(2, 9, 3, torch.float32, dev="cpu"))
    for rev in (False, True):
        xs, gs, hs = (t.clone().requires_grad_() for t in (x, g, h0))
        s, rows = hs, [None] * 9
        for t in (range(8, -1, -1) if rev else range(9)):
            s = torch.sigmoid(gs[:, t]) * s + (1 - torch.sigmoid(gs[:, t])) * xs[:, t]
            rows[t] = s
        want = torch.autograd.grad([torch.stack(rows, 1), s], [xs, gs, hs], [dh, dlast])
        o = oracle(x, g, h0, dh, dlast, rev)
        for k, w in zip(("dx", "dg", "dh0"), want):
            assert float((o[k][0] - w).abs().max()) < 1e-12


def test_refusals_on_cpu():
    from unet_amd import _lib, ops
    x, g = torch.zeros(2, 4, 6), torch.zeros(2, 4, 6)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.gated_scan(x, g)
    with pytest.raises(ValueError, match="must both be"):
        ops.gated_scan(x, g[:, :3])
    with pytest.raises(ValueError, match="must both be"):
        ops.gated_scan(x[0], g[0])
    with pytest.raises(TypeError, match="one dtype"):
        ops.gated_scan(x, g.bfloat16())
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.gated_scan(x.half(), g.half())
    with pytest.raises(ValueError, match="state must be"):
        ops.gated_scan(x, g, torch.zeros(2, 5))
    with pytest.raises(TypeError, match="state must be float32"):
        ops.gated_scan(x, g, torch.zeros(2, 6, dtype=torch.float64))
    with pytest.raises(ValueError, match="must both be"):
        ops.gated_scan_step(x, g, torch.zeros(2, 6))
    with pytest.raises(ValueError, match="state must be"):
        ops.gated_scan_step(x[0], g[0], torch.zeros(3, 6))
    with pytest.raises(RuntimeError, match="no backward"):
        ops.gated_scan_step(x[0], g[0].requires_grad_(), torch.zeros(4, 6))
    lib = _lib.load()
    for ld in (-1, (1 << 22) + 1):
        assert lib.unet_gated_scan_fwd(0, 16, 0, ld, 16, 0, 1, None, 0, 1, 2, 1, 16, None, None, None, 0, None) == -1
        assert b"row pitch" in lib.unet_last_error()
        assert lib.unet_gated_scan_bwd(0, 16, 0, 1, 16, 0, 1, 16, 16, 0, ld, None, 0, 1, 2, 1, 16, 16, None, None, 0, None) == -1
        assert b"row pitch" in lib.unet_last_error()
    assert lib.unet_gated_scan_fwd(0, None, 0, 0, None, 0, 0, None, 0, 1, 1, 1, None, None, None, None, 0, None) == -1
    assert b"null" in lib.unet_last_error()
    assert lib.unet_gated_scan_fwd(7, 16, 0, 0, 16, 0, 0, None, 0, 1, 1, 1, 16, None, None, None, 0, None) == -1
    assert b"dtype" in lib.unet_last_error()
    assert lib.unet_gated_scan_fwd(0, 16, 0, 0, 16, 0, 0, None, 0, 1, 0, 1, 16, None, None, None, 0, None) == -1
    assert b"shape" in lib.unet_last_error()
    # one long sequence is split into segments and needs its workspace
    need = lib.unet_gated_scan_workspace_bytes(0, 1, 100000, 64)
    assert need > 0
    assert lib.unet_gated_scan_fwd(0, 16, 0, 64, 16, 0, 64, None, 0, 1, 100000, 64, 16, None, None, None, 0, None) == -1
    assert b"workspace" in lib.unet_last_error()
    assert lib.unet_gated_scan_bwd(0, 16, 0, 64, 16, 0, 64, 16, 16, 0, 64, None, 0, 1, 100000, 64, 16, 16, None, 16, need - 8, None) == -1
    assert b"workspace" in lib.unet_last_error()
    assert lib.unet_gated_scan_step(0, None, 0, None, 0, None, None, 1, 1, None) == -1
    assert lib.unet_gated_scan_workspace_bytes(0, 64, 1024, 1024) == 0


# ------------------------------------------------------------------------------------------------ GPU
SHAPES = [(1, 1, 1), (2, 1, 130), (3, 2, 7), (1, 63, 2), (2, 64, 64), (2, 65, 66), (5, 333, 199), (3, 129, 128), (64, 40, 96),
          (1, 5000, 36), (2, 2111, 257), (300, 70, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,l,c", SHAPES)
def test_values_and_gradients(n, l, c, dtype):
    for reverse, state in ((False, True), (True, True), (False, False)):
        x, g, h0, dh, dlast = inputs(n, l, c, dtype, seed=n + l)
        h0, dlast = (h0, dlast) if state else (None, None)
        got = call(x, g, h0, dh, dlast, reverse)
        want = oracle(x, g, h0, dh, dlast, reverse)
        for k in got:
            near(got[k], want[k], (k, reverse, state))
        assert got["h"].dtype == dtype and got["last"].dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_alignment_and_broadcast(dtype):
    """Column ranges of one projection, at even and odd offsets; every second row; one window broadcast over the batch."""
    n, l, c = 3, 150, 66
    x, g, h0, dh, dlast = inputs(n, l, 2 * c + 5, dtype, seed=4)
    for a, b in ((0, c), (1, c + 2), (2, c + 5)):
        xs, gs, d = x[:, :, a:a + c], g[:, :, b:b + c], dh[:, :, a:a + c]
        got, want = call(xs, gs, h0[:, :c].contiguous(), d, None, False), oracle(xs, gs, h0[:, :c], d, None, False)
        for k in got:
            near(got[k], want[k], (k, a, b))
    xs, gs, d = x[:, ::2, :c], g[:, 1::2, :c], dh[:, ::2, :c]
    got, want = call(xs, gs, None, d, None, True), oracle(xs, gs, None, d, None, True)
    for k in got:
        near(got[k], want[k], (k, "rows"))
    one = x[:1, :, :c].contiguous().requires_grad_()
    from unet_amd import ops
    gs, d = g[:, :, :c], dh[:, :, :c]
    h = ops.gated_scan(one.expand(n, l, c), gs)
    want = oracle(one.detach().expand(n, l, c), gs, None, d, None, False)
    near(h, want["h"], "broadcast")
    (dx,) = torch.autograd.grad(h, one, d)
    half = torch.finfo(dtype).eps / 2      # each window's gradient is rounded before the sum, the sum once more
    value, bound = want["dx"]
    tol = (bound + half * value.abs()).sum(0) + 4 * half * value.abs().sum(0)
    assert bool(((dx[0].double().cpu() - value.sum(0)).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saturated_gates(dtype):
    """Gates of +-inf and +-1e4: the state passes unchanged, or is replaced, and no gradient reaches the gate."""
    from unet_amd import ops
    x, g, h0, dh, dlast = inputs(2, 200, 64, dtype, seed=5)
    for big in (float("inf"), 1e4):
        got = call(x, torch.full_like(g, big), h0, dh, dlast, False)
        assert torch.equal(got["h"], h0[:, None].expand(2, 200, 64).to(dtype)) and torch.equal(got["last"], h0)
        assert float(got["dx"].abs().max()) == 0 and float(got["dg"].abs().max()) == 0
        want = dlast.double() + dh.double().sum(1)
        assert float((got["dh0"].double() - want).abs().max()) <= 200 * U * float(dh.double().abs().sum(1).max())
        got = call(x, torch.full_like(g, -big), h0, dh, dlast, False)
        assert torch.equal(got["h"], x) and torch.equal(got["last"], x[:, -1].float())
        assert float(got["dg"].abs().max()) == 0 and float(got["dh0"].abs().max()) == 0
    # a NaN stays in its window and channel, in the rows behind it
    x[0, 100, 3] = float("nan")
    h = ops.gated_scan(x, g)
    assert bool(torch.isnan(h[0, 100:, 3]).any()) and int(torch.isnan(h).sum()) == int(torch.isnan(h[0, 100:, 3]).sum())
    assert not bool(torch.isnan(h[0, :100]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_and_single_rows_continue_each_other(dtype):
    from unet_amd import ops
    x, g, h0, _, _ = inputs(3, 150, 70, dtype, seed=6)
    want = oracle(x, g, h0, None, None, False)
    a, s = ops.gated_scan(x[:, :101], g[:, :101], h0, return_state=True)
    b, s = ops.gated_scan(x[:, 101:140], g[:, 101:140], s, return_state=True)
    rows = [ops.gated_scan_step(x[:, t], g[:, t], s) for t in range(140, 150)]
    near(torch.cat([a, b, torch.stack(rows, 1)], 1), want["h"], "pieces")
    near(s, want["last"], "state")
    empty, last = ops.gated_scan(x[:, :0], g[:, :0], h0, return_state=True)
    assert empty.shape == (3, 0, 70) and torch.equal(last, h0)
    assert ops.gated_scan(x[:0], g[:0]).shape == (0, 150, 70)
    with pytest.raises(ValueError, match="contiguous"):
        ops.gated_scan_step(x[:, 0], g[:, 0], torch.zeros(70, 3, device="cuda").t())


@pytest.mark.gpu
def test_partial_gradients_and_differences():
    """Only the final state used; only some inputs want a gradient; a directional difference quotient."""
    from unet_amd import ops
    x, g, h0, dh, dlast = inputs(2, 90, 32, torch.float32, seed=7)
    xr = x.clone().requires_grad_()
    _, last = ops.gated_scan(xr, g, h0, return_state=True)
    (dx,) = torch.autograd.grad(last, xr, dlast)
    near(dx, oracle(x, g, h0, torch.zeros_like(dh), dlast, False)["dx"], "last only")
    hr = h0.clone().requires_grad_()
    (d0,) = torch.autograd.grad(ops.gated_scan(x, g, hr), hr, dh)
    near(d0, oracle(x, g, h0, dh, None, False)["dh0"], "h0 only")
    got = call(x, g, h0, dh, dlast, True)
    dirs = [torch.randn_like(t) for t in (x, g, h0)]
    eps = 2.0 ** -7

    def loss(sign):
        h, last = ops.gated_scan(*(t + sign * eps * d for t, d in zip((x, g, h0), dirs)), reverse=True, return_state=True)
        return float((h.double() * dh.double()).sum() + (last.double() * dlast.double()).sum())

    want = sum(float((got[k].double() * d.double()).sum()) for k, d in zip(("dx", "dg", "dh0"), dirs))
    quotient = (loss(1) - loss(-1)) / (2 * eps)
    # third-order remainder eps^2 / 6 * |f'''| of a sum over 5760 outputs of unit size, and rounding 1e-7 / eps of the same sum
    assert abs(quotient - want) <= (eps ** 2 + 1e-6 / eps) * (float(dh.abs().sum()) + abs(want))


@pytest.mark.gpu
def test_side_stream_and_graph_replays():
    from unet_amd import ops
    x, g, h0, dh, dlast = inputs(2, 700, 40, torch.bfloat16, seed=8)
    eager = call(x, g, h0, dh, dlast, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(x, g, h0, dh, dlast, False)
    side.synchronize()
    for k in eager:
        assert torch.equal(eager[k], other[k]), k
    del other
    xs, gs = x.clone().requires_grad_(), g.clone().requires_grad_()
    state = h0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, last = ops.gated_scan(xs, gs, h0, return_state=True)
        dx, dg = torch.autograd.grad([h, last], [xs, gs], [dh, dlast])
        row = ops.gated_scan_step(xs.detach()[:, 0], gs.detach()[:, 0], state)
    want_state = h0.clone()
    for rep in range(4):
        x2, g2, _, _, _ = inputs(2, 700, 40, torch.bfloat16, seed=20 + rep)
        with torch.no_grad():
            xs.copy_(x2)
            gs.copy_(g2)
        graph.replay()
        torch.cuda.synchronize()
        want = call(x2, g2, h0, dh, dlast, False)
        want_row = ops.gated_scan_step(x2[:, 0], g2[:, 0], want_state)
        for a, b in ((h, want["h"]), (last, want["last"]), (dx, want["dx"]), (dg, want["dg"]), (row, want_row), (state, want_state)):
            assert torch.equal(a, b), rep


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """2.2e9 elements: the last window's rows lie past 2^31 elements and 2^32 bytes."""
    from unet_amd import ops
    n, l, c = 3, 700000, 1024
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((n, l, c), generator=gen, device="cuda", dtype=torch.bfloat16)
    g = torch.randn((n, l, c), generator=gen, device="cuda", dtype=torch.bfloat16)
    h, last = ops.gated_scan(x, g, return_state=True)
    cut = slice(l - 300, l)
    state = torch.zeros(1, c)          # 300 rows behind an unknown state: sigmoid(g) products have long forgotten it
    want = oracle(x[2:, cut], g[2:, cut], state, None, None, False)
    near(h[2:, -100:], tuple(v[:, -100:] for v in want["h"]), "tail")
    near(last[2:], want["last"], "last")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pitch,l", [(1 << 22, 130), ((1 << 22) + 6, 3)])
def test_row_pitches_up_to_and_past_the_descriptor(pitch, l, dtype):
    """2^22 elements a row is what a tile's 32-bit offsets reach; a longer pitch is copied."""
    c = 6
    x, g, h0, dh, dlast = inputs(1, l, c, dtype, seed=11)
    wide = []
    for t in (x, g, dh):
        w = torch.empty((l - 1) * pitch + c, dtype=dtype, device="cuda").as_strided((1, l, c), (0, pitch, 1))
        wide.append(w.copy_(t))
    for rev in (False, True):
        got = call(wide[0], wide[1], h0, wide[2], dlast, rev)
        want = oracle(x, g, h0, dh, dlast, rev)
        for k in got:
            near(got[k], want[k], (k, rev))


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    from unet_amd import ops
    x, g, h0, dh, _ = inputs(1, 70, 8, torch.float32, seed=12)
    x.requires_grad_()
    h = ops.gated_scan(x, g, h0)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(h, x, dh, create_graph=True)


@pytest.mark.gpu
def test_two_captured_graphs_in_turn():
    """Split rows (workspace) in two graphs that replay on two streams at once and in turn, with eager work between."""
    from unet_amd import ops
    sets = [inputs(1, 3000 + 50 * i, 40, torch.bfloat16, seed=13 + i)[:3] for i in range(2)]
    graphs, outs = [], []
    for x, g, h0 in sets:
        ops.gated_scan(x, g, h0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.gated_scan(x, g, h0, return_state=True))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for x, g, h0 in sets:
            g.add_(0.25)
        torch.cuda.synchronize()
        if rep % 2:
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        else:
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for (x, g, h0), (h, last) in zip(sets, outs):
            h2, last2 = ops.gated_scan(x, g, h0, return_state=True)
            assert torch.equal(h, h2) and torch.equal(last, last2), rep


def check_moved_state(dev):
    from unet_amd import ops
    w, state = torch.ones(2, 8, device=dev, requires_grad=True), torch.full((2, 8), 2.0, device=dev)
    loss = (w * state[:]).sum()                 # saves the state (a view of it) for backward
    version = state._version
    with torch.no_grad():
        ops.gated_scan_step(torch.ones(2, 8, device=dev), torch.zeros(2, 8, device=dev), state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_moved_state_is_seen_by_autograd_on_cpu(monkeypatch):
    from unet_amd import ops
    monkeypatch.setattr(ops, "_run", lambda *a: None)
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    check_moved_state("cpu")


@pytest.mark.gpu
def test_a_moved_state_is_seen_by_autograd():
    check_moved_state("cuda")


# ---------------------------------------------------------------------------------------- long memories
def long_gates(c):
    """Gates from 9 to 18.6, a constant per channel; half of them put 1 - sigmoid halfway between two multiples of 2^-24, where
    rounding the gate itself to 32 bits would be furthest off."""
    k = torch.logspace(0, 3.2, c // 2, dtype=torch.float64).floor()
    keep = (k + 0.5) * U
    return torch.cat([torch.linspace(9.0, 18.6, c - c // 2, dtype=torch.float64), torch.log((1 - keep) / keep)]).float()


def long_oracle(x, g, h0, dh, dlast):
    """As ``oracle``, for a kernel whose states keep 1 - f: a row's gate costs keep times a relative error (400 u: 40 u of the gate, and
    the chains of up to 200 pairs that span a long sequence), and the state itself is rounded once per 8 rows (a span of 8 rows is
    one step of the state's chain) and 16 units more on the way to a row (8 rows, each a rounding and half a unit of the rounded
    gate, and the last step).  The adjoint likewise; sums of dh over a span of up to
    12288 rows round in steps of at least 192 rows: 100 u |dh| a row."""
    x, g, d = (t.double().cpu() for t in (x, g, dh))
    s, mu = h0.double().cpu(), dlast.double().cpu()
    e, em = torch.zeros_like(s), torch.zeros_like(s)
    f, keep = torch.sigmoid(g), torch.sigmoid(-g)
    l, top = x.shape[1], d.abs().amax(1)
    h, eh, before, eb, dx, ex, dg, eg = (torch.empty_like(x) for _ in range(8))
    for t in range(l):
        before[:, t], eb[:, t] = s, e + 16 * U * s.abs()
        e = f[:, t] * e + 400 * U * keep[:, t] * (s.abs() + x[:, t].abs())
        s = f[:, t] * s + keep[:, t] * x[:, t]
        e += U / 8 * s.abs()
        h[:, t], eh[:, t] = s, e + 16 * U * s.abs()
    last = (s, e + 16 * U * s.abs())
    for t in range(l - 1, -1, -1):
        lam = d[:, t] + mu
        el = em + 16 * U * lam.abs()
        diff, ed = before[:, t] - x[:, t], eb[:, t] + U * (before[:, t].abs() + x[:, t].abs())
        fk = f[:, t] * keep[:, t]
        dx[:, t], ex[:, t] = keep[:, t] * lam, keep[:, t] * (el + 2 * K * U * lam.abs())
        dg[:, t], eg[:, t] = lam * diff * fk, fk * (el * diff.abs() + lam.abs() * ed + 3 * K * U * (lam * diff).abs())
        mu = f[:, t] * lam
        em = f[:, t] * em + 400 * U * keep[:, t] * lam.abs() + U / 8 * mu.abs() + 100 * U * top
    return dict(h=(h, eh), last=last, dx=(dx, ex), dg=(dg, eg), dh0=(mu, em + 16 * U * mu.abs()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,l", [(1, 20000), (300, 3000)])
def test_long_memories(n, l, dtype):
    """Split sequences and whole ones, with gates whose memory is 8 thousand to 120 million rows."""
    c = 64
    gen = torch.Generator().manual_seed(l)
    r = lambda *s: 1.0 + 0.3 * torch.randn(*s, generator=gen)
    x, dh, h0, dlast = r(n, l, c).to(dtype).cuda(), r(n, l, c).to(dtype).cuda(), r(n, c).cuda(), r(n, c).cuda()
    g = long_gates(c).to(dtype).cuda().expand(n, l, c)
    got, want = call(x, g, h0, dh, dlast, False), long_oracle(x, g, h0, dh, dlast)
    for k in got:
        near(got[k], want[k], k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_constant_input_holds_its_state(dtype):
    """x = h0 is the recurrence's fixed point, whatever the gate.  A span's A + B / x differs from 1 by the roundings of its sums, at most
    2.5 R + 5 units of C for a chain of R, and a state leaves a fixed point only where that exceeds half an ulp (C above 1 / 40), to
    come back at a rate of C: 2.5 R + 5 + 100 units, R at most 200.  A single row's f + rest + keep is 1 to one rounding."""
    from unet_amd import ops
    v = torch.linspace(1.0, 1.9375, 64).to(dtype).float().cuda()
    v[::2] *= -1
    for n, l in ((1, 75000), (300, 3000)):
        g = long_gates(64).to(dtype).cuda().expand(n, l, 64)
        for reverse in (False, True):
            h, last = ops.gated_scan(v.to(dtype).expand(n, l, 64), g, v.expand(n, 64), reverse=reverse, return_state=True)
            assert float((last.double() / v.double() - 1).abs().max()) <= 605 * U, (n, l, reverse)
    state, x = v.repeat(3, 1), v.to(dtype).repeat(3, 1)
    g = torch.stack([long_gates(64), -long_gates(64), torch.linspace(-9, 9, 64)]).to(dtype).cuda()
    for _ in range(3000):
        ops.gated_scan_step(x, g, state)
    assert float((state.double() / v.double() - 1).abs().max()) <= 2 * U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_inputs_stay_infinite(dtype):
    """An infinite input makes its state infinite for the rest of the sequence, of one sign, without a NaN where gates are open."""
    from unet_amd import ops
    for n, l in ((1, 5000), (300, 130)):
        x, g, h0, _, _ = inputs(n, l, 64, dtype, seed=40)
        g = g.abs() + 0.5
        g[:, :, 32:] += 12.0
        x[0, 70, 3], x[0, 70, 40] = float("inf"), -float("inf")
        h, last = ops.gated_scan(x, g, h0, return_state=True)
        assert not bool(torch.isnan(h).any())
        assert bool((h[0, 70:, 3] == float("inf")).all()) and bool((h[0, 70:, 40] == -float("inf")).all())
        assert int(torch.isinf(h).sum()) == 2 * (l - 70) and int(torch.isinf(last).sum()) == 2
        state = last.clone()
        ops.gated_scan_step(x[:, 0], g[:, 0], state)
        assert torch.equal(torch.isinf(state), torch.isinf(last)) and not bool(torch.isnan(state).any())


def one_row_views(dev, dtype):
    """[N, 1, C] whose only row has a stride of 2^23, and [1, C] and [N, C] rows that far apart: views of what a caller holds."""
    c, far = 8, 1 << 23
    rows = torch.randn(2 * far, generator=torch.Generator().manual_seed(0)).to(dtype).to(dev)
    return rows.as_strided((3, 1, c), (c, far, 1)), rows.as_strided((2, c), (far, 1)), rows.as_strided((1, c), (far, 1))


def test_strides_of_an_only_row_are_ignored_on_cpu(monkeypatch):
    """Neither refused (a transposed [1, N, C] has such a stride) nor copied; single rows go in as they are, whatever lies between them."""
    from unet_amd import ops
    calls = []
    monkeypatch.setattr(ops, "_run", lambda *a: calls.append(a))
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    wide, rows, one = one_row_views("cpu", torch.float32)
    ops.gated_scan(wide, wide)
    assert calls[0][3:9] == (wide.data_ptr(), 8, 8, wide.data_ptr(), 8, 8)
    for x in (rows, one):
        ops.gated_scan_step(x, x, torch.zeros(x.shape))
        assert calls[-1][3:7] == (x.data_ptr(), 1 << 23, x.data_ptr(), 1 << 23)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_of_an_only_row(dtype):
    from unet_amd import ops
    wide, rows, one = one_row_views("cuda", dtype)
    state, dlast = torch.randn(2, 3, 8, generator=torch.Generator().manual_seed(1)).cuda()
    got, want = call(wide, wide, state, wide, dlast, True), oracle(wide, wide, state, wide, dlast, True)
    # dh passes the gate rounded to 32 bits, dlast the span's a + rest: half an ulp of the gate apart, u relative, which shows where
    # the two cancel and the bound of their sum does not cover it
    want["dh0"] = (want["dh0"][0], want["dh0"][1] + U * wide[:, 0].double().cpu().abs())
    for k in got:
        near(got[k], want[k], k)
    for x in (rows, one):
        s = state[:x.shape[0]].clone()
        h = ops.gated_scan_step(x, x, s)
        w = oracle(x[:, None], x[:, None], state[:x.shape[0]], None, None, False)
        near(h[:, None], w["h"], "row")
        near(s, w["last"], "state")


def test_sizes_past_the_librarys_counters_are_refused_on_cpu(monkeypatch):
    """2^32 + 5 rows are not 5 rows, and a launch holds 2^32 threads."""
    from unet_amd import _lib, ops
    monkeypatch.setattr(ops, "_run", lambda *a: pytest.fail("called"))
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    for shape in ((1, (1 << 32) + 5, 1), ((1 << 32) + 5, 1, 1)):
        x = torch.zeros(1).expand(shape)
        with pytest.raises(ValueError, match="below 2\\^31"):
            ops.gated_scan(x, x)
    x, state = torch.zeros(1).expand(1 << 31, 1), torch.zeros(1).expand(1 << 31, 1)
    with pytest.raises(ValueError, match="below 2\\^31"):
        ops.gated_scan_step(x, x, state)
    for shape in ((1, (1 << 32) + 8, 8), ((1 << 32) + 1, 1, 8)):
        q = torch.zeros(1).expand(shape)
        with pytest.raises(ValueError, match="below 2\\^31"):
            ops.rel_bias_attention(q, q, q, torch.zeros(8, 1), 1, max_distance=5)
    lib = _lib.load()
    for dtype, n in ((1, 1 << 23), (0, 1 << 23)):
        assert lib.unet_gated_scan_fwd(dtype, 16, 1, 1, 16, 1, 1, None, 0, n, 1, 1, 16, None, None, None, 0, None) == -1
        assert b"2^32 threads" in lib.unet_last_error()
        assert lib.unet_gated_scan_bwd(dtype, 16, 1, 1, 16, 1, 1, 16, 16, 1, 1, None, 0, n, 1, 1, 16, 16, None, None, 0, None) == -1
        assert b"2^32 threads" in lib.unet_last_error()
        assert lib.unet_gated_scan_step(dtype, 16, 1 << 20, 16, 1 << 20, 16, 16, 1 << 12, 1 << 20, None) == -1
        assert b"2^32 threads" in lib.unet_last_error()
        st = (C.c_int32 * 2)(0, 1)
        rows = 129 if dtype == 0 else 65
        assert lib.unet_rel_attn_fwd(dtype, 16, 16, 16, 16, 1, 4, st, None, 65535, rows, 2048, 256, 1.0, 16, None, None, None, 0, None) == -1
        assert b"workgroups" in lib.unet_last_error()


@pytest.mark.gpu
def test_rows_up_to_the_last_int():
    """2^31 - 4097 rows in 512 segments: the last one would end past 2^31 if it were whole.  Checked where it begins (backward
    passes its adjoint on) and where it ends."""
    from unet_amd import ops
    l = 2 ** 31 - 4097
    gen = torch.Generator(device="cuda").manual_seed(41)
    x, g, dh = (torch.randn((1, l, 1), generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    h, last = ops.gated_scan(x.requires_grad_(), g.requires_grad_(), return_state=True)
    dx, dg = torch.autograd.grad(h, (x, g), dh)
    for mid, hi in ((511 * 65536 * 64, 511 * 65536 * 64 + 300), (l - 200, l)):
        cut = slice(mid - 600, hi)             # 300 rows on either side forget what lies beyond them
        want = oracle(x.detach()[:, cut], g.detach()[:, cut], None, dh[:, cut], None, False)
        inner = slice(300, 700 if hi < l else None)
        for k, t in (("h", h), ("dx", dx), ("dg", dg)):
            near(t[:, cut][:, inner], tuple(v[:, inner] for v in want[k]), (k, mid))
    near(last, want["last"], "last")
