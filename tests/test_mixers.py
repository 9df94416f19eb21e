"""The bottleneck layers built on the new operators (RelativeSelfAttention1D, GatedRecurrence1D), alone against torch in
float64, inside CondUNet1D, and trained with the 8-bit optimizer: the operators together, as a user runs them."""
import pytest
import torch

import unet_amd


# ------------------------------------------------------------------------------------------------ CPU
def test_construction_and_refusals_on_cpu():
    for kind, cls in (("relative", unet_amd.RelativeSelfAttention1D), ("recurrent", unet_amd.GatedRecurrence1D)):
        m = unet_amd.CondUNet1D(base=32, conv_type="modern", attention_type=kind, activation="gelu")
        assert any(isinstance(x, cls) for x in m.mid) and m.get_attention_module() is None
        again = unet_amd.CondUNet1D(base=32, conv_type="modern", attention_type=kind, activation="gelu")
        again.load_state_dict(m.state_dict(), strict=True)
    with pytest.raises(ValueError, match="multiple of 8"):
        unet_amd.RelativeSelfAttention1D(36)
    with pytest.raises(ValueError, match="buckets"):
        unet_amd.RelativeSelfAttention1D(64, n_buckets=7)
    with pytest.raises(ValueError, match="whole window"):
        unet_amd.GatedRecurrence1D(16).forward_step(torch.zeros(1, 16), torch.zeros(1, 16))
    # a plain module's checkpoint loads but for the table, which starts at zero
    rel, plain = unet_amd.RelativeSelfAttention1D(64), unet_amd.SelfAttention1D(64)
    missing, unexpected = rel.load_state_dict(plain.state_dict(), strict=False)
    assert missing == ["rel_table"] and not unexpected and float(rel.rel_table.detach().abs().max()) == 0
    from unet_amd.trainer import Trainer
    with pytest.raises(ValueError, match="native"):
        Trainer(torch.nn.Linear(2, 2), optimizer="torch", state_bits=8, compute_dtype=None)


# ------------------------------------------------------------------------------------------------ GPU
def _conv(m, x):
    return x @ m.weight[:, :, 0].T + m.bias


def _relative64(m, x):
    from unet_amd import ops
    q, k, v = (_conv(c, x) for c in (m.query, m.key, m.value))
    l, heads = x.shape[1], m.rel_table.shape[1]
    pos = torch.arange(l, device=x.device)
    bias = m.rel_table[ops.rel_bucket(pos[None, :] - pos[:, None], m.rel_table.shape[0], m.max_distance)]
    hd = x.shape[2] // heads
    outs = [torch.softmax(q @ k.transpose(1, 2).contiguous() + bias[..., h], -1) @ v[..., h * hd:(h + 1) * hd] for h in range(heads)]
    return x + m.gamma * torch.cat(outs, -1)


def _recurrent64(m, x):
    hs = []
    for i, (vm, fm) in enumerate(zip(m.value, m.forget)):
        v, f = _conv(vm, x), torch.sigmoid(_conv(fm, x))
        s, rows = torch.zeros_like(x[:, 0]), [None] * x.shape[1]
        for t in (reversed(range(x.shape[1])) if i else range(x.shape[1])):
            s = f[:, t] * s + (1 - f[:, t]) * v[:, t]
            rows[t] = s
        hs.append(torch.stack(rows, 1))
    return x + m.gamma * _conv(m.out_proj, torch.cat(hs, -1))


def _module(kind, c, seed=0, **kw):
    torch.manual_seed(seed)
    m = (unet_amd.RelativeSelfAttention1D if kind == "relative" else unet_amd.GatedRecurrence1D)(c, **kw)
    with torch.no_grad():
        m.gamma.fill_(0.7)
        if kind == "relative":
            m.rel_table.normal_()
            m.query.weight.mul_(2.0)
    return m.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,kw", [("relative", {}), ("recurrent", {}), ("recurrent", dict(bidirectional=False))])
@pytest.mark.parametrize("l", [1, 100, 203])
def test_layers_against_float64(kind, kw, l):
    """fp32 kernels against the formula in float64.  A value passes at most four products of 64..128 terms and the mixing in
    between, each within (terms + 40) u of its terms' magnitudes; gradients twice that.  Magnitudes grow to about ten times the
    result's rms in a cancelling sum: 4 * 168 * 2^-24 * 10 = 4e-4 of the result's largest value."""
    c = 64
    m = _module(kind, c, **kw)
    ref = _module(kind, c, **kw).double()
    x = torch.randn(2, c, l, device="cuda")
    w = torch.randn_like(x)
    xa, xb = x.clone().requires_grad_(), x.double().transpose(1, 2).contiguous().requires_grad_()
    out = m(xa)
    want = (_relative64 if kind == "relative" else _recurrent64)(ref, xb)
    (out * w).sum().backward()
    (want * w.double().transpose(1, 2)).sum().backward()

    def close(a, b, what, tol=4e-4):
        assert float((a.double() - b).abs().max()) <= tol * float(b.abs().max()) + 1e-9, what

    close(out.detach(), want.detach().transpose(1, 2), "out")
    close(xa.grad, xb.grad.transpose(1, 2), "dx", 8e-4)
    # a parameter's gradient is a sum over 2 l rows whose terms partly cancel: the bound is of the sum's terms, 8e-4 of the largest
    # entry of the module's gradients of that kind
    for (name, p), q in zip(m.named_parameters(), ref.parameters()):
        scale = max(float(q.grad.abs().max()), 1e-2 * float(xb.grad.abs().max()))
        assert float((p.grad.double() - q.grad).abs().max()) <= 8e-4 * scale * max(1.0, l ** 0.5 / 10) + 1e-9, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_table_equals_plain_attention(dtype):
    rel, plain = _module("relative", 128), unet_amd.SelfAttention1D(128).cuda()
    plain.load_state_dict({k: v for k, v in rel.state_dict().items() if k != "rel_table"})
    with torch.no_grad():
        rel.rel_table.zero_()
        x = torch.randn(2, 128, 300, device="cuda").to(dtype)
        a, b = rel(x).float(), plain(x).float()
    # the two kernels round the same probabilities and outputs once each: two half steps of the attention's output and of the sum
    half = torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 2e-6
    assert float((a - b).abs().max()) <= 4 * half * float(b.abs().max())


@pytest.mark.gpu
def test_padded_batch_and_rows_one_by_one():
    m = _module("relative", 64)
    x = torch.randn(3, 120, 64, device="cuda")
    lengths = torch.tensor([120, 0, 77], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        got = m.forward_nlc(x, lengths)
        assert torch.equal(got[1], x[1]) and torch.equal(got[2, 77:], x[2, 77:])
        short = m.forward_nlc(x[2:, :77].contiguous())
        assert float((got[2, :77] - short[0]).abs().max()) <= 1e-5 * float(short.abs().max())
        r = _module("recurrent", 64, bidirectional=False).eval()
        for dtype, tol in ((torch.float32, 1e-5), (torch.bfloat16, 4 * 2.0 ** -8)):
            xs = x.to(dtype)
            whole = r.forward_nlc(xs)
            state = torch.zeros(3, 64, device="cuda")
            rows = torch.stack([r.forward_step(xs[:, t], state) for t in range(120)], 1)
            assert float((rows.float() - whole.float()).abs().max()) <= tol * float(whole.float().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["relative", "recurrent"])
def test_training_run_with_8bit_moments(kind):
    """CondUNet1D with the layer in its bottleneck, bf16, trained by Trainer(state_bits=8): eager steps and the captured step give
    the same parameters, the state is in 8 bits, and a checkpoint continues the run bit by bit."""
    from unet_amd.optim import ClipAdamW
    from unet_amd.trainer import Trainer

    def build(use_graph):
        torch.manual_seed(3)
        model = unet_amd.CondUNet1D(in_channels=8, out_channels=8, base=32, emb_dim=16, conv_type="modern", attention_type=kind,
                                    activation="gelu").cuda()
        with torch.no_grad():
            model.outc.weight.normal_(0, 0.02)
            model.mid[2].gamma.fill_(0.5)
        return model, Trainer(model, state_bits=8, use_graph=use_graph, nan_check_every=1000)

    gen = torch.Generator().manual_seed(4)
    batches = [(torch.randn(4, 8, 1100, generator=gen).cuda(), torch.randint(0, 7, (4,), generator=gen).cuda(),
                torch.randn(4, 8, 1100, generator=gen).cuda()) for _ in range(4)]
    eager_model, eager = build(False)
    graph_model, graphed = build(True)
    assert isinstance(eager.opt, ClipAdamW)
    start = [p.detach().clone() for p in eager_model.parameters()]
    ob, ids, tgt = batches[0]
    for _ in range(3):                       # the captured trainer takes three warm-up steps on its first batch
        eager.step(ob, tgt, ids)
    for ob, ids, tgt in batches:
        for tr in (eager, graphed):
            loss = tr.step(ob, tgt, ids)
            assert bool(torch.isfinite(loss.detach()))
    moved = 0
    for (name, a), b, s in zip(eager_model.named_parameters(), graph_model.parameters(), start):
        assert torch.equal(a, b), name
        moved += int(not torch.equal(a, s))
    assert moved >= len(start) - 2
    mixer = [p for p in eager_model.mid[2].parameters()]
    assert all(p.grad is None or bool(torch.isfinite(p.grad).all()) for p in mixer)
    assert eager.opt.state[mixer[0]]["exp_avg"].dtype == (torch.float8_e4m3fn if mixer[0].numel() >= 4096 else torch.float32)
    big = [p for p in eager_model.parameters() if p.numel() >= 4096]
    assert big and all(eager.opt.state[p]["exp_avg"].dtype == torch.float8_e4m3fn for p in big)
    # checkpoint
    import copy
    saved = copy.deepcopy((eager_model.state_dict(), eager.opt.state_dict()))
    other_model, other = build(False)
    other_model.load_state_dict(saved[0])
    other.opt.load_state_dict(saved[1])
    ob, ids, tgt = batches[0]
    eager.step(ob, tgt, ids)
    other.step(ob, tgt, ids)
    for (name, a), b in zip(eager_model.named_parameters(), other_model.parameters()):
        assert torch.equal(a, b), name


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bidirectional", [False, True])
def test_recurrence_alone_follows_its_optimizer(bits, bidirectional):
    """A module of its own, in the mode it is born in: every call without gradients sees the weights of the last step (the native
    optimizer writes them without telling their version counters), as does an eval() after it."""
    from unet_amd.optim import ClipAdamW
    m = _module("recurrent", 64, bidirectional=bidirectional)
    opt = ClipAdamW(m.parameters(), lr=0.05, state_bits=bits)
    x = torch.randn(2, 64, 50, device="cuda")

    def calls(mod):
        with torch.no_grad():
            out = [mod(x)]
            if not bidirectional:
                state = torch.zeros(2, 64, device="cuda")
                out += [mod.forward_step(x[:, :, 0], state), state]
        return out

    for it in range(4):
        if it == 3:
            m.eval()
        fresh = _module("recurrent", 64, seed=1, bidirectional=bidirectional)
        fresh.load_state_dict(m.state_dict())
        for a, b in zip(calls(m), calls(fresh)):
            assert torch.equal(a, b), it
        opt.zero_grad()
        m(x).square().sum().backward()
        opt.step()
