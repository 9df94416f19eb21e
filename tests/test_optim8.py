"""optim.ClipAdamW with 8-bit moments (csrc/optim8.hip): refusals and the storage format on the CPU, steps on the GPU against
float64.

A step from given codes is compared value by value.  With u = 2^-24: m and v are sums of two products (5 roundings with the
clip, and a fast reciprocal and square root of 2 units each in the update), so the stored value before its rounding is within
8 u relative of the terms' magnitudes, and the parameter within u of itself plus 16 u of the step.  The stored code is the
nearest of that value: at most half a step, 2^-4 relative or 2^-10 of the smallest code's unit, from the exact value, plus the
8 u (which may move a value across a border to the other neighbour, still within half a step of the value it rounds)."""
import copy
import math

import pytest
import torch

U = 2.0 ** -24
BETAS = (0.7595905764360957, 0.920298282605139)      # train.py:186-188
BLOCK = 256


def e4m3(y):
    """Nearest e4m3 value of a float64 tensor, ties to even."""
    _, ex = torch.frexp(y)
    step = torch.exp2((ex - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


# ------------------------------------------------------------------------------------------------ CPU
def test_storage_format_on_cpu():
    from unet_amd.optim import FP8_LEAST, dequantise_moment, quantise_moment
    gen = torch.Generator().manual_seed(0)
    for n in (1, 255, 256, 257, 4096, 5000):
        x = torch.randn(n, generator=gen) * 10.0 ** torch.randint(-6, 3, (n,), generator=gen)
        codes, scale = quantise_moment(x, False)
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scale.shape == (-(-n // BLOCK),)
        back = dequantise_moment(codes, scale).double()
        per = scale.double().repeat_interleave(BLOCK)[:n]
        assert bool(((back - x.double()).abs() <= (2.0 ** -4 * x.double().abs()).clamp_min(2.0 ** -10 * per) * (1 + 1e-6)).all())
        # codes of codes: unchanged
        codes2, scale2 = quantise_moment(back.float(), False)
        assert torch.allclose(dequantise_moment(codes2, scale2), back.float(), rtol=3e-7, atol=0)
    r = torch.tensor([1.0, 1e-9, 0.0] + [0.5] * 253)
    codes, scale = quantise_moment(r, True)
    assert codes[:3].float().tolist() == [448.0, FP8_LEAST, 0.0]        # a positive root stays positive
    for tiny in (0.0, 1e-31, 1e-45):                                     # far below any eps: zeros, no overflowing 448 / max
        codes, scale = quantise_moment(torch.full((300,), tiny), True)
        assert float(codes.float().abs().max()) == 0 and float(scale.abs().max()) == 0


def test_refusals_on_cpu():
    from unet_amd import _lib
    from unet_amd.optim import ClipAdamW
    p = torch.nn.Parameter(torch.zeros(5000))
    for kw in (dict(state_bits=16), dict(state_bits=8, min_8bit_numel=-1), dict(betas=(1.0, 0.9))):
        with pytest.raises(ValueError):
            ClipAdamW([p], **kw)
    opt = ClipAdamW([p], state_bits=8)
    with pytest.raises(ValueError, match="state_bits"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3))], "state_bits": 4})
    assert len(opt.param_groups) == 1
    with pytest.raises(TypeError, match="fp32"):
        ClipAdamW([torch.nn.Parameter(torch.zeros(5000, dtype=torch.bfloat16))], state_bits=8).moment_buffers()
    from unet_amd.optim import _dense_fp32
    dense = torch.zeros(3, 4)
    assert _dense_fp32([dense, None]) and _dense_fp32([None]) and _dense_fp32([])
    for bad in (dense.to_sparse(), dense.to_sparse_csr(), dense.t(), dense.bfloat16()):
        assert not _dense_fp32([dense, bad])
    lib = _lib.load()
    assert lib.unet_adamw8_apply(None, 1, None, None, None, None, 1, None, None, None, None, None, None, None, None, None, 0.9, 0.9,
                                 1e-8, 0.0, None) == -1 and b"null" in lib.unet_last_error()
    assert lib.unet_adamw8_prepare(None, 0, None, 0, 0, 5.0, 16, 16, None, 0.9, 0.9, None, None) == -1
    assert b"clip" in lib.unet_last_error()
    assert lib.unet_adamw8_prepare(None, 300, None, 0, 0, 0.0, 16, 16, 16, 0.9, 0.9, 16, None) == -1
    assert b"at most" in lib.unet_last_error()
    assert lib.unet_adamw8_sqnorm(None, 1, 16, 16, 1, 16, None) == -1 and b"null" in lib.unet_last_error()
    assert [lib.unet_adamw8_norm_blocks(b) for b in (1, 32, 33, 16384)] == [1, 1, 2, 512]
    assert [lib.unet_adamw8_blocks(b) for b in (1, 4, 5, 16384)] == [1, 1, 2, 4096]


def test_partly_stepped_groups_keep_their_moments_on_cpu():
    """A loaded group of which some large tensors have codes, one fp32 moments and one nothing yet."""
    from unet_amd.optim import ClipAdamW, dequantise_moment, quantise_moment
    gen = torch.Generator().manual_seed(1)
    params = [torch.nn.Parameter(torch.zeros(s)) for s in ((50, 100), (4097,), (5000,), (10,))]
    m, v = torch.randn(50, 100, generator=gen), torch.rand(50, 100, generator=gen)
    codes = dict(zip(("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale"),
                     quantise_moment(m, False) + quantise_moment(v.sqrt(), True)))
    m2, v2 = torch.randn(5000, generator=gen), torch.rand(5000, generator=gen)
    opt = ClipAdamW(params, state_bits=8)
    saved = opt.state_dict()
    saved["state"] = {0: dict(codes, step=torch.tensor(3.0)), 2: dict(exp_avg=m2, exp_avg_sq=v2, step=torch.tensor(7.0))}
    opt.load_state_dict(copy.deepcopy(saved))
    opt.moment_buffers()
    st = opt.state[params[0]]
    for k, t in codes.items():
        assert torch.equal(st[k].float(), t.float()), k
    assert [float(opt.state[p]["step"]) for p in params] == [3, 0, 7, 0]
    st = opt.state[params[2]]
    want = quantise_moment(m2, False)
    assert torch.equal(dequantise_moment(st["exp_avg"], st["exp_avg_scale"]), dequantise_moment(*want))
    for i in (1, 3):
        assert float(opt.state[params[i]]["exp_avg"].float().abs().max()) == 0


# ------------------------------------------------------------------------------------------------ GPU
SHAPES = [(256, 32, 7), (256,), (1,), (3,), (512, 256, 1), (37, 5), (1024, 130), (2, 3, 5, 7), (8193,), (4096,), (4095,), (90, 99),
          (0,), (4096, 33)]


def make(seed=0, shapes=SHAPES, unaligned=()):
    gen = torch.Generator().manual_seed(seed)
    params = []
    for i, s in enumerate(shapes):
        t = torch.randn(*s, generator=gen)
        if i in unaligned:      # storage that starts 4 bytes behind a 16-byte boundary
            buf = torch.empty(t.numel() + 1, device="cuda")
            v = buf[1:].view(t.shape)
            v.copy_(t)
            params.append(torch.nn.Parameter(v))
        else:
            params.append(torch.nn.Parameter(t.cuda()))
    return params, gen


def set_grads(params, gen, scale):
    for i, p in enumerate(params):
        g = torch.randn(p.shape, generator=gen) * scale * 10.0 ** (-(i % 4))
        g *= torch.rand(p.shape, generator=gen) > 0.1
        p.grad = g.cuda()


def snapshot(opt, params):
    """Every tensor's moments as float64 values, and what they are held in."""
    from unet_amd.optim import _load_moments
    out = []
    for p in params:
        st = opt.state[p]
        m, v = (t.double() for t in _load_moments(st))
        out.append((m.view(p.shape), v.view(p.shape), "exp_avg_scale" in st, float(st["step"])))
    return out


def check_step(opt, params, before_p, before, grads, lr, wd, max_norm, eps=1e-8):
    b1, b2 = BETAS
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads if g is not None))
    assert abs(float(opt.total_norm()) - norm) <= 2e-6 * norm
    clip = min(1.0, max_norm / (norm + 1e-6)) if max_norm else 1.0
    for p, p0, (m0, v0, small, t0), g, (m1, v1, _, t1) in zip(params, before_p, before, grads, snapshot(opt, params)):
        if g is None:
            assert torch.equal(p, p0) and torch.equal(m0, m1) and torch.equal(v0, v1) and t0 == t1
            continue
        if not p.numel():
            continue
        assert t1 == t0 + 1
        g = g.double() * clip
        ma, mb, v = b1 * m0, (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        m = ma + mb
        step = lr * (m / (1 - b1 ** t1)) / ((v / (1 - b2 ** t1)).sqrt() + eps)
        want = p0.double() * (1 - lr * wd) - step
        size = lr * ((ma.abs() + mb.abs()) / (1 - b1 ** t1)) / ((v / (1 - b2 ** t1)).sqrt() + eps)
        # the clip's norm is a float of fp32 partial sums: 2e-6 relative, which only the clipped gradient sees
        rel = 16 * U + (2e-6 if max_norm else 0.0)
        tol = 3 * U * p0.double().abs() + rel * size + 1e-37
        assert bool(((p.double() - want).abs() <= tol).all()), float(((p.double() - want).abs() / tol).max())
        near = 8 * U + (2e-6 if max_norm else 0.0)
        if not small:
            assert bool(((m1 - m).abs() <= near * (ma.abs() + mb.abs()) + 1e-45).all())
            assert bool(((v1 - v).abs() <= 2 * near * v + 1e-45).all())
            continue
        r = v.sqrt()
        for stored, x, mag in ((m1, m, ma.abs() + mb.abs()), (v1.sqrt(), r, r)):
            flat = torch.nn.functional.pad(x.reshape(-1).abs(), (0, -x.numel() % BLOCK)).view(-1, BLOCK)
            unit = (flat.amax(1) / 448).repeat_interleave(BLOCK)[:x.numel()].view(x.shape)      # one code unit of the block
            half = torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * unit)
            err = (stored - x).abs()
            ok = err <= half * (1 + 1e-5) + near * mag
            if x is r:           # a positive root below half the smallest code is raised to it
                ok |= (x > 0) & (x < 2.0 ** -9 * unit) & (err <= 2.0 ** -9 * unit * (1 + 1e-5))
                assert bool(((stored > 0) == (x > 0)).all() | (unit < 1e-30).any())
            assert bool(ok.all()), float((err / half).max())
            # and it is the nearest code: nearly all equal a rounding done in float64
            if float(unit.min()) > 0:
                near_all = e4m3(x / unit)
                if x is r:
                    near_all = torch.where((x > 0) & (near_all == 0), torch.full_like(near_all, 2.0 ** -9), near_all)
                differ = ((stored / unit - near_all).abs() > 1e-4 * near_all.abs()).double().mean()
                # a value lies within `near` of a border with probability 2 * near * 2^4 at most: allow ten times that, plus one
                assert float(differ) <= 320 * near + 1.0 / x.numel() + 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm,scale", [(5.0, 30.0), (5.0, 1e-4), (None, 1.0)])
@pytest.mark.parametrize("wd", [0.0, 0.01])
def test_steps_match_float64(max_norm, scale, wd):
    from unet_amd.optim import ClipAdamW
    params, gen = make(0, unaligned=(0, 8))
    opt = ClipAdamW(params, lr=2e-3, betas=BETAS, weight_decay=wd, max_grad_norm=max_norm, state_bits=8)
    opt.moment_buffers()
    for it in range(4):
        set_grads(params, gen, scale)
        if it == 2:
            params[0].grad = params[3].grad = None
        if it == 3:        # a gradient whose storage is not 16-byte aligned
            g = params[6].grad
            buf = torch.empty(g.numel() + 1, device="cuda")
            buf[1:] = g.reshape(-1)
            params[6].grad = buf[1:].view(g.shape)
        grads = [None if p.grad is None else p.grad.clone() for p in params]
        p0, before = [p.detach().clone() for p in params], snapshot(opt, params)
        opt.step()
        check_step(opt, params, p0, before, grads, 2e-3, wd, max_norm)
        for p, g in zip(params, grads):
            assert g is None or torch.equal(p.grad, g)
    buf = opt.moment_buffers()
    assert buf["exp_avg8"].dtype == torch.float8_e4m3fn and buf["exp_avg8"].numel() == 256 * buf["exp_avg8_scale"].numel()
    small = [p for p in params if p.numel() < 4096]
    assert all("exp_avg_sq" in opt.state[p] for p in small) and not any("exp_avg_sq" in opt.state[p] for p in params if p.numel() >= 4096)


@pytest.mark.gpu
def test_extreme_gradients():
    """Zero, tiny and huge gradients stay finite; an infinite one spoils its own block of 256 only."""
    from unet_amd.optim import ClipAdamW
    p = torch.nn.Parameter(torch.ones(8192, device="cuda"))
    opt = ClipAdamW([p], lr=1e-3, betas=BETAS, weight_decay=0.0, state_bits=8)
    g = torch.zeros(8192, device="cuda")
    g[256:512] = 1e-38
    g[512:768] = 1e18
    g[768:1024] = torch.logspace(-12, 3, 256, device="cuda")
    for _ in range(5):
        p.grad = g.clone()
        opt.step()
        assert bool(torch.isfinite(p).all())
        assert float((p - 1).detach().abs().max()) <= 5 * 1e-3 * 3      # no step is blown up by a vanished root
    assert torch.equal(p[:256], torch.ones(256, device="cuda")) and torch.equal(p[1024:], torch.ones(7168, device="cuda"))
    g[2000] = float("inf")
    p.grad = g
    opt.step()
    p.grad = torch.zeros_like(g)
    opt.step()
    bad = ~torch.isfinite(p)
    lo = 2000 // 256 * 256
    assert bool(bad[2000]) and not bool(bad[:lo].any()) and not bool(bad[lo + 256:].any())


@pytest.mark.gpu
def test_checkpoints_convert_both_ways():
    from unet_amd.optim import ClipAdamW, _load_moments
    shapes = [(64, 64, 3), (7,), (100, 50)]
    params, gen = make(3, shapes)
    opt = ClipAdamW(params, lr=1e-3, betas=BETAS, weight_decay=0.0, state_bits=8, max_grad_norm=1.0)
    for _ in range(3):
        set_grads(params, gen, 1.0)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    assert saved["state"][0]["exp_avg"].dtype == torch.float8_e4m3fn and saved["state"][1]["exp_avg"].dtype == torch.float32
    set_grads(params, gen, 1.0)
    grads = [p.grad.clone() for p in params]
    start = [p.detach().clone() for p in params]
    opt.step()
    # 8 -> 8: the same trajectory to the bit
    other = [torch.nn.Parameter(s.clone()) for s in start]
    opt2 = ClipAdamW(other, lr=1e-3, betas=BETAS, weight_decay=0.0, state_bits=8, max_grad_norm=1.0)
    opt2.load_state_dict(saved)
    for p, g in zip(other, grads):
        p.grad = g.clone()
    opt2.step()
    for a, b in zip(params, other):
        assert torch.equal(a, b)
        assert set(opt.state[a]) == set(opt2.state[b])
        for k, x in opt.state[a].items():
            assert x.dtype == opt2.state[b][k].dtype and torch.equal(x.float(), opt2.state[b][k].float()), k
    # 8 -> 32: the values the codes stand for
    third = [torch.nn.Parameter(s.clone()) for s in start]
    opt3 = ClipAdamW(third, lr=1e-3, betas=BETAS, weight_decay=0.0, max_grad_norm=1.0)
    opt3.load_state_dict(saved)
    assert opt3.param_groups[0]["state_bits"] == 32
    opt3.moment_buffers()
    for i, p in enumerate(third):
        m, v = _load_moments(saved["state"][i])
        assert torch.equal(opt3.state[p]["exp_avg"].reshape(-1), m.cuda()) and torch.equal(opt3.state[p]["exp_avg_sq"].reshape(-1), v.cuda())
        assert set(opt3.state[p]) == {"step", "exp_avg", "exp_avg_sq"} and float(opt3.state[p]["step"]) == 3
    # torch's AdamW -> 8
    ref = torch.optim.AdamW(third, lr=1e-3, betas=BETAS, weight_decay=0.0)
    for p, g in zip(third, grads):
        p.grad = g.clone()
    ref.step()
    opt4 = ClipAdamW(third, lr=1e-3, betas=BETAS, weight_decay=0.0, state_bits=8, max_grad_norm=2.0)
    opt4.load_state_dict(copy.deepcopy(ref.state_dict()))
    assert opt4.param_groups[0]["state_bits"] == 8 and opt4.param_groups[0]["max_grad_norm"] == 2.0
    opt4.moment_buffers()
    m, v = _load_moments(opt4.state[third[0]])
    want = ref.state[third[0]]
    top = float(want["exp_avg"].abs().max())
    assert float((m - want["exp_avg"].reshape(-1)).abs().max()) <= 2.0 ** -4 * top
    assert float((v.sqrt() - want["exp_avg_sq"].reshape(-1).sqrt()).abs().max()) <= 2.0 ** -4 * float(want["exp_avg_sq"].max().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [1.0, None])
def test_graph_replays_and_many_tensors(max_norm):
    """300 tensors (two sub-tables) in a captured step: every replay equals an eager optimizer's step, lr read from memory."""
    from unet_amd.optim import ClipAdamW
    shapes = [(40 + i, 110) if i % 3 else (17 + i,) for i in range(300)]
    a, gen = make(5, shapes)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    lr = torch.tensor(1e-3, device="cuda")
    kw = dict(betas=BETAS, weight_decay=0.01, max_grad_norm=max_norm, state_bits=8)
    eager, cap = ClipAdamW(a, lr=1e-3, **kw), ClipAdamW(b, lr=lr, **kw)
    for p in b:
        p.grad = torch.zeros_like(p)
    cap.moment_buffers()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.step()
    for rep in range(4):
        set_grads(a, gen, 1.0)
        for p, q in zip(a, b):
            q.grad.copy_(p.grad)
        if rep == 2:
            lr.fill_(5e-4)
            eager.param_groups[0]["lr"] = 5e-4
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), rep
        assert torch.equal(eager.total_norm(), cap.total_norm())
    for x, y in zip(eager.moment_buffers().values(), cap.moment_buffers().values()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.gpu
def test_thawed_tensors_and_switched_state_bits():
    """A frozen tensor joins after some steps; then the group goes to fp32 moments and back: nobody's moments are lost."""
    from unet_amd.optim import ClipAdamW
    params, gen = make(6, [(64, 80), (70, 90), (9,)])
    lr, wd = 1e-2, 0.01
    opt = ClipAdamW(params, lr=lr, betas=BETAS, weight_decay=wd, state_bits=8, max_grad_norm=5.0)
    params[1].requires_grad_(False)
    for _ in range(2):
        set_grads(params, gen, 1.0)
        params[1].grad = None
        opt.step()
    fresh = lambda p, small: (torch.zeros_like(p, dtype=torch.float64), torch.zeros_like(p, dtype=torch.float64), small, 0.0)
    a, c = snapshot(opt, [params[0], params[2]])
    before = [a, fresh(params[1].detach(), True), c]
    params[1].requires_grad_(True)
    for bits in (8, 32):
        opt.param_groups[0]["state_bits"] = bits
        before = [(m, v, bits == 8 and p.numel() >= 4096, t) for (m, v, _, t), p in zip(before, params)]
        set_grads(params, gen, 1.0)
        p0 = [p.detach().clone() for p in params]
        opt.step()
        after = snapshot(opt, params)
        assert [small for _, _, small, _ in after] == [bits == 8, bits == 8, False]
        check_step(opt, params, p0, before, [p.grad for p in params], lr, wd, 5.0)
        before = after
    opt.param_groups[0]["state_bits"] = 8
    set_grads(params, gen, 0.0)
    opt.step()
    for (m, v, _, _), (m1, v1, small, t), p in zip(before, snapshot(opt, params), params):
        assert small == (p.numel() >= 4096) and t == (3 if p is params[1] else 5)
        # the moments are rounded to codes once on the way in and once when the step stores them
        assert float((m1 - BETAS[0] * m).abs().max()) <= 2 * 2.0 ** -4 * float(m.abs().max())
        assert float((v1.sqrt() - (BETAS[1] * v).sqrt()).abs().max()) <= 2 * 2.0 ** -4 * float(v.max().sqrt())


@pytest.mark.gpu
def test_checkpoint_files(tmp_path):
    """8-bit state through a checkpoint file, read without unpickling anything but tensors: the next step has the same bits."""
    from unet_amd.checkpoint import load_checkpoint, save_checkpoint
    from unet_amd.optim import ClipAdamW
    torch.manual_seed(0)
    nets = [torch.nn.Linear(90, 77).cuda() for _ in range(2)]
    opts = [ClipAdamW(net.parameters(), lr=1e-2, betas=BETAS, state_bits=8, max_grad_norm=1.0) for net in nets]
    gen = torch.Generator().manual_seed(8)
    for _ in range(2):
        set_grads(list(nets[0].parameters()), gen, 1.0)
        opts[0].step()
    save_checkpoint(nets[0], opts[0], 2, tmp_path / "c.pt")
    load_checkpoint(tmp_path / "c.pt", nets[1], optimizer=opts[1])
    set_grads(list(nets[0].parameters()), gen, 1.0)
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        q.grad = p.grad.clone()
    for opt in opts:
        opt.step()
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, q)
        for k, t in opts[0].state[p].items():
            assert torch.equal(t.float(), opts[1].state[q][k].float()), k


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_gradient_norms_that_are_not_finite(bad):
    """With a clip the norm carries a NaN to every tensor, and an infinite norm takes the other gradients to zero, as
    clip_grad_norm_ in front of torch's AdamW does; the fp32 tensors of the group likewise."""
    from unet_amd.optim import ClipAdamW
    shapes = [(40, 130), (77,), (5000,), (3,)]
    params, gen = make(9, shapes)
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    kw = dict(lr=1e-3, betas=BETAS, weight_decay=0.0)
    opt, ref = ClipAdamW(params, max_grad_norm=1.0, state_bits=8, **kw), torch.optim.AdamW(other, **kw)
    for it in range(2):
        set_grads(params, gen, 1.0)
        if it == 1:
            params[2].grad[1234] = bad
        for p, q in zip(params, other):
            q.grad = p.grad.clone()
        before = [p.detach().clone() for p in params]
        opt.step()
        torch.nn.utils.clip_grad_norm_(other, 1.0)
        ref.step()
    block = torch.zeros(5000, dtype=torch.bool, device="cuda")
    block[1234 // 256 * 256:1234 // 256 * 256 + 256] = True      # shares the spoilt element's scale
    for i, (p, q, p0) in enumerate(zip(params, other, before)):
        stray = torch.isnan(p) != torch.isnan(q)
        assert not bool((stray & ~block if i == 2 else stray).any()), i
        if math.isinf(bad):       # the first step's momentum alone: lr m / sqrt(v) changes, by less than a few steps of lr
            keep = torch.isfinite(p)
            assert int((~keep).sum()) == (1 if i == 2 else 0)
            assert 0 < float((p - p0)[keep].abs().max()) < 4e-3
        else:
            assert bool(torch.isnan(p).all())


def check_changed_threshold(dev, step):
    """min_8bit_numel of a group that has its tables: the next step, or the next look at its buffers, goes by the new value, and
    no moment is lost on the way."""
    from unet_amd.optim import ClipAdamW
    gen = torch.Generator().manual_seed(2)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dev)) for s in ((50, 100), (3000,), (10,))]
    opt = ClipAdamW(params, lr=1e-3, betas=BETAS, weight_decay=0.0, state_bits=8)
    opt.moment_buffers()
    step(opt, params, gen)
    for numel, coded in ((2048, (True, True, False)), (6000, (False, False, False)), (0, (True, True, True)), (4096, (True, False, False))):
        before = snapshot(opt, params)
        opt.param_groups[0]["min_8bit_numel"] = numel
        assert opt.moment_buffers()["exp_avg8"].numel() == sum(-(-p.numel() // BLOCK) * BLOCK for p, c in zip(params, coded) if c)
        after = snapshot(opt, params)
        assert tuple(small for _, _, small, _ in after) == coded
        for p, (m, v, _, t), (m1, v1, _, t1) in zip(params, before, after):
            assert t == t1
            flat = torch.nn.functional.pad(torch.stack([m, v.sqrt()]).view(2, -1).abs(), (0, -p.numel() % BLOCK)).view(2, -1, BLOCK)
            half = 2.0 ** -4 * flat.amax(2).repeat_interleave(BLOCK, 1)[:, :p.numel()].view(2, *p.shape)
            assert bool(((m1 - m).abs() <= half[0]).all()) and bool(((v1.sqrt() - v.sqrt()).abs() <= half[1]).all())
        step(opt, params, gen)
        assert tuple(small for _, _, small, _ in snapshot(opt, params)) == coded


def test_a_changed_threshold_takes_effect_on_cpu():
    def step(opt, params, gen):                 # no kernel here: moments written as a loaded state would be
        for p in params:
            st = opt.state[p]
            if "exp_avg_sq" in st:
                st["exp_avg"].copy_(torch.randn(p.shape, generator=gen))
                st["exp_avg_sq"].copy_(torch.rand(p.shape, generator=gen))
    check_changed_threshold("cpu", step)


@pytest.mark.gpu
def test_a_changed_threshold_takes_effect():
    def step(opt, params, gen):
        set_grads(params, gen, 1.0)
        opt.step()
    check_changed_threshold("cuda", step)


def check_loaded_codes(dev):
    """A loaded state is what the checkpoint holds: e4m3 codes at one byte an element, also before the first step; the checkpoint itself is
    left alone, and a second one saved from it is the same."""
    from unet_amd.optim import ClipAdamW, quantise_moment
    gen = torch.Generator().manual_seed(3)
    params = [torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((50, 100), (8192,), (10,))]
    opt = ClipAdamW(params, state_bits=8)
    saved = opt.state_dict()
    names = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
    saved["state"] = {i: dict(zip(names, quantise_moment(torch.randn(s, generator=gen), False) +
                                  quantise_moment(torch.rand(s, generator=gen), True)), step=torch.tensor(4.0))
                      for i, s in enumerate(((50, 100), (8192,)))}
    keep = copy.deepcopy(saved)
    for bits in (8, 32):
        opt = ClipAdamW(params, state_bits=bits)
        opt.load_state_dict(saved)
        again = opt.state_dict()
        for i in (0, 1):
            assert set(saved["state"][i]) == set(keep["state"][i]) == set(again["state"][i])
            for k, t in keep["state"][i].items():
                for got in (saved["state"][i][k], again["state"][i][k], opt.state[params[i]][k]):
                    assert got.dtype == t.dtype and torch.equal(got.cpu().float(), t.float()), k
                if k != "step":
                    assert opt.state[params[i]][k].device == params[i].device
        buf = opt.moment_buffers()
        if bits == 8:
            assert torch.equal(buf["exp_avg8"][5120:].cpu().view(torch.uint8), keep["state"][1]["exp_avg"].view(torch.uint8))
    # codes that an earlier load had cast to fp32 on their way into a file
    for st in saved["state"].values():
        for k in ("exp_avg", "exp_avg_sq_root"):
            st[k] = st[k].float()
    opt = ClipAdamW(params, state_bits=8)
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[params[0]]["exp_avg"].cpu().view(torch.uint8), keep["state"][0]["exp_avg"].view(torch.uint8))


def test_loaded_codes_keep_their_type_on_cpu():
    check_loaded_codes("cpu")


@pytest.mark.gpu
def test_loaded_codes_keep_their_type():
    check_loaded_codes("cuda")


def step_in_torch(p, g, codes, lr, wd, clip, t):
    """One step of a tensor from its codes in 32-bit torch operations, in the kernel's order: (parameter, codes, scales, size of the
    parameter's step).  The bias corrections are 64-bit numbers rounded once."""
    from unet_amd.optim import dequantise_moment
    b1, b2 = BETAS
    f32 = lambda v: torch.tensor(v, dtype=torch.float64, device=p.device).float()
    pad = lambda x: torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    m, r = (pad(dequantise_moment(*codes[i:i + 2])) for i in (0, 2))
    gc = pad(g) * clip
    m = m * f32(b1) + gc * f32(1 - b1)
    r = torch.sqrt(r * r * f32(b2) + gc * f32(1 - b2) * gc)
    out = []
    for x in (m, r):
        top = x.abs().amax(1, keepdim=True)
        y = x * ((1.0 / top) * 448.0)
        if x is r:
            y = torch.where(r > 0, y.clamp_min(2.0 ** -9), y)
        out += [y.to(torch.float8_e4m3fn).view(-1)[:p.numel()].view(p.shape), (top * f32(1 / 448).item()).view(-1)]
    step = f32(lr / (1 - b1 ** t)) * (m / (r * f32(1 / math.sqrt(1 - b2 ** t)) + 1e-8))
    return p * (1 - f32(lr) * f32(wd)) - step.view(-1)[:p.numel()].view(p.shape), out, step.view(-1)[:p.numel()].view(p.shape)


def clip_of(grads, max_norm, ulps=0):
    """(norm, clip) with the squares summed in 64 bits, and the norm moved by some units in its last place."""
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    for _ in range(ulps):
        norm = torch.nextafter(norm, torch.full_like(norm, math.inf))
    return norm, torch.clamp(max_norm * (1.0 / (norm + 1e-6)), max=1.0)


def test_codes_show_an_ulp_of_the_norm_on_cpu():
    """What the next test compares is sensitive enough: with a norm a few units off in its last place, as a sum in 32 bits may leave it,
    some of 2 M codes differ."""
    gen = torch.Generator().manual_seed(4)
    g = torch.randn(2 ** 21, generator=gen)
    zero = [torch.zeros(2 ** 21).to(torch.float8_e4m3fn), torch.zeros(2 ** 13)] * 2
    a, b = (step_in_torch(torch.zeros(2 ** 21), g, zero, 1e-3, 0.0, clip_of([g], 1.0, ulps)[1], 1)[1] for ulps in (0, 2))
    assert any(int((x.view(torch.uint8) != y.view(torch.uint8)).sum()) > 0 for x, y in ((a[0], b[0]), (a[2], b[2])))
    assert not torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm,wd", [(1.0, 0.01), (1e6, 0.0)])
def test_a_clipped_step_has_the_bits_of_32_bit_torch(max_norm, wd):
    """Codes and scales to the bit, the norm as the rounding of its 64-bit sum; a parameter differs by single roundings.  The step:
    here the root's product, + eps, the division and the product with lr / (1 - b1^t), 4 u; there one fma, a reciprocal of one unit (2 u), two
    products, 5 u; and lr is rounded there before it is divided, and both quotients are, 3 u: 12 u.  p keep - step: either side
    rounds 1 - lr wd (together u), the product and the difference (u each on either side): 5 u of the larger of p before and after."""
    from unet_amd.optim import ClipAdamW
    params, gen = make(11, [(1024, 1030), (300, 7, 129), (4097,), (512, 512, 7)])
    opt = ClipAdamW(params, lr=2e-3, betas=BETAS, weight_decay=wd, max_grad_norm=max_norm, state_bits=8)
    opt.moment_buffers()
    names = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
    for t in (1, 2, 3):
        set_grads(params, gen, 0.3)
        norm, clip = clip_of([p.grad for p in params], max_norm)
        old = [p.detach().clone() for p in params]
        want = [step_in_torch(p.detach().clone(), p.grad, [opt.state[p][k].clone() for k in names], 2e-3, wd, clip, t) for p in params]
        opt.step()
        assert torch.equal(opt.total_norm(), norm)
        for p, p0, (p1, codes, step) in zip(params, old, want):
            for k, x in zip(names, codes):
                got = opt.state[p][k]
                assert torch.equal(got.view(torch.uint8), x.view(torch.uint8)), (t, k, int((got.float() != x.float()).sum()))
            off, size = (p.detach().double() - p1.double()).abs(), torch.maximum(p0.double().abs(), p1.double().abs())
            assert float((off - 5 * U * size - 12 * U * step.double().abs()).max()) <= 0


@pytest.mark.gpu
def test_a_state_loaded_before_its_parameters_moved():
    """A checkpoint loaded beside parameters on the CPU that then move to the device: the codes follow at the next look or step."""
    from unet_amd.optim import ClipAdamW, quantise_moment
    gen = torch.Generator().manual_seed(6)
    net = torch.nn.Linear(90, 77)
    opt = ClipAdamW(net.parameters(), state_bits=8)
    saved = opt.state_dict()
    codes = quantise_moment(torch.randn(77, 90, generator=gen), False) + quantise_moment(torch.rand(77, 90, generator=gen), True)
    names = ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
    saved["state"] = {0: dict(zip(names, codes), step=torch.tensor(2.0))}
    opt.load_state_dict(saved)
    net.cuda()
    opt.moment_buffers()
    for k, t in zip(names, codes):
        got = opt.state[net.weight][k]
        assert got.is_cuda and torch.equal(got.cpu().view(torch.uint8), t.view(torch.uint8)), k
    for p in net.parameters():
        p.grad = torch.zeros_like(p)
    opt.step()
    assert float(opt.state[net.weight]["step"]) == 3
