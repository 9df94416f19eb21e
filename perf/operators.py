"""Cases for measuring the framework's sequence and optimizer operators: the gated linear recurrence, attention with a
learned relative-position bias, and the AdamW step with 8-bit moments.

``own`` selects what ``run`` computes: False, the operators' plain forms (elementary torch operations in 32 bits, rounded
once at the end); True, the calls a user makes of ``unet_amd``.  ``exact`` evaluates the definitions in 64 bits.
"""
import math

import torch

own = False

BETAS = (0.7595905764360957, 0.920298282605139)     # the trainer's defaults
BLOCK = 256                                          # elements that share one scale of the 8-bit moments
FP8_MAX = 448.0                                      # largest e4m3 value
SMALL = 4096                                         # tensors with fewer elements keep 32-bit moments

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one new row for a handful of live recordings: a real-time decoder calls this once per sample, so latency counts
        dict(name="scan_step_live", op="scan_step", n=8, c=512, dtype="bf16"),
        # the bottleneck of the default training configuration: 64 windows, 4096 samples / 4, base 256 * 4 channels
        dict(name="scan_train_bottleneck", op="scan", n=64, l=1024, c=1024, dtype="bf16", train=True, reverse=False,
             state=False, strided=False),
        # a 300 s recording at 1 kHz as one sequence through the same bottleneck: few sequences, a long axis
        dict(name="scan_infer_recording", op="scan", n=1, l=75000, c=1024, dtype="bf16", train=False, reverse=False,
             state=True, strided=False),
        # parity runs in fp32: the backward direction of a bidirectional layer, odd sizes, row-strided inputs, carried state
        dict(name="scan_train_odd_fp32", op="scan", n=5, l=333, c=199, dtype="fp32", train=True, reverse=True, state=True,
             strided=True),
        # attention over one short window of a narrow model: launch-bound
        dict(name="rel_infer_window", op="rel", n=1, l=64, c=64, heads=8, buckets=32, distance=128, dtype="bf16",
             train=False, ragged=False, local=False),
        # the bottleneck attention of the default configuration in training
        dict(name="rel_train_bottleneck", op="rel", n=32, l=1024, c=1024, heads=8, buckets=32, distance=128, dtype="bf16",
             train=True, ragged=False, local=False),
        # one long recording segment, most of whose pairs lie in the two outermost buckets
        dict(name="rel_infer_long", op="rel", n=1, l=8192, c=512, heads=8, buckets=32, distance=128, dtype="bf16",
             train=False, ragged=False, local=False),
        # parity runs in fp32: padded batch (one window with no valid position), far pairs switched off by -inf, odd length
        dict(name="rel_train_odd_fp32", op="rel", n=3, l=301, c=160, heads=4, buckets=16, distance=50, dtype="fp32",
             train=True, ragged=True, local=True),
        # a small model of the hyper-parameter search: launch-bound
        dict(name="adam8_narrow", op="adam", base=16, down=2, kernel=3, branches=1, io=32, clip=5.0, decay=0.0),
        # the constructor's default width and convolutions
        dict(name="adam8_default", op="adam", base=128, down=2, kernel=3, branches=1, io=32, clip=0.0, decay=0.01),
        # the training default (base 256, four dilated branches of 7 taps)
        dict(name="adam8_training", op="adam", base=256, down=2, kernel=7, branches=4, io=32, clip=5.0, decay=0.0),
        # the wide model: 128 channels in and out, four downsampling stages
        dict(name="adam8_wide", op="adam", base=256, down=4, kernel=7, branches=4, io=128, clip=5.0, decay=0.01),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_step", "rel", "rel", "adam"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "scan_step":
        return dict(op=op, n=_log(rng, 1, 256), c=_log(rng, 8, 4096), dtype=dtype)
    if op == "scan":
        n, c = _log(rng, 1, 128), _log(rng, 4, 2048)
        most = 64 * 1024 * 1024 // (1 if dtype == "bf16" else 2)
        l = min(_log(rng, 1, 75000), max(1, most // (n * c)))
        return dict(op=op, n=n, l=l, c=c, dtype=dtype, train=rng.random() < 0.6, reverse=rng.random() < 0.5,
                    state=rng.random() < 0.5, strided=rng.random() < 0.3)
    if op == "rel":
        heads = rng.choice([1, 2, 4, 8])
        hd = 8 * rng.randint(1, 32) if dtype == "bf16" else 4 * rng.randint(1, 32)
        train = rng.random() < 0.6
        l = _log(rng, 1, 2048 if dtype == "bf16" else 512)
        most = 16 * (1 << 30) if dtype == "bf16" else 1 << 30                  # multiply-adds of q k^T
        n = min(_log(rng, 1, 32), max(1, most // (l * l * heads * hd)))
        buckets = 4 * rng.randint(1, 16)
        distance = rng.randint(buckets // 4 + 1, 512)
        return dict(op=op, n=n, l=l, c=heads * hd, heads=heads, buckets=buckets, distance=distance, dtype=dtype,
                    train=train, ragged=rng.random() < 0.4, local=rng.random() < 0.3)
    kernel, branches = rng.choice([(3, 1), (7, 4)])
    return dict(op=op, base=_log(rng, 8, 256), down=rng.randint(1, 3), kernel=kernel, branches=branches,
                io=rng.randint(1, 64), clip=rng.choice([0.0, 5.0]), decay=rng.choice([0.0, 0.01]))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(case):
    """Valid positions of every window of a padded batch: from none to all."""
    n, l = case["n"], case["l"]
    return [l] if n == 1 else [(l * i) // (n - 1) for i in range(n)]


def _starts(buckets, distance):
    """starts[b]: the smallest |offset| of bucket b of one side.  Half of a side's buckets hold one distance each, the
    others grow geometrically up to ``distance``; exact integer arithmetic, so no border depends on a rounded log."""
    side, exact_ = buckets // 2, buckets // 4
    m = side - exact_
    out = list(range(exact_))
    a = exact_
    for k in range(m):
        while a ** m * exact_ ** k < distance ** k * exact_ ** m:
            a += 1
        out.append(a)
    return out


def _param_shapes(case):
    """The parameter list of the framework's U-Net at these settings."""
    base, down, k, br, io, emb = case["base"], case["down"], case["kernel"], case["branches"], case["io"], 128
    ch = [base] + [min(base * 2 ** (i + 1), base * 8) for i in range(down)]
    out = [(7, emb)]

    def block(ci, co):
        got = []
        for _ in range(br):
            got += [(co, ci, k), (co,)]
        got += [(co,), (co,)]
        if br > 1:
            r = max(co // 4, 8)
            got += [(br,), (r, co), (co, r)]
        return got + [(co, co, 1), (co,), (co, emb), (co,), (co, emb), (co,), (co, co, 1), (co,), (co, emb), (co,)]

    out += block(io, ch[0])
    for i in range(down):
        out += block(ch[i], ch[i + 1])
    for i in range(down):
        ci, co = ch[down - i], ch[down - i - 1]
        out += [(ci, co, 4), (co,)] + block(co, co)
    out += [(ch[down], ch[down], 3), (ch[down],)] * 2 + [(io, ch[0], 3), (io,)]
    return out


def _layout(case):
    """(shape, region, first element) per tensor; region 8 starts at multiples of BLOCK, region 32 at multiples of 4."""
    end, rows = {8: 0, 32: 0}, []
    for s in _param_shapes(case):
        n = math.prod(s)
        region, pad = (8, BLOCK) if n >= SMALL else (32, 4)
        rows.append((s, region, end[region]))
        end[region] += -(-n // pad) * pad
    return rows, end


def _quantise(x):
    """x [blocks, BLOCK] -> e4m3 codes and one fp32 scale per block; a positive value never becomes zero if x >= 0."""
    top = x.abs().amax(1, keepdim=True)
    scale = top / FP8_MAX
    inv = torch.where(top > 0, FP8_MAX / top, torch.zeros_like(top))
    return (x * inv).to(torch.float8_e4m3fn), scale.squeeze(1)


def _prepare_adam(case, seed):
    g = _gen(seed)
    rows, end = _layout(case)
    flat = {}
    for region in (8, 32):
        n = end[region]
        used = torch.zeros(n, device="cuda")
        size = torch.ones(n, device="cuda")
        for i, (s, reg, a) in enumerate(rows):
            if reg == region:
                used[a:a + math.prod(s)] = 1.0
                size[a:a + math.prod(s)] = 10.0 ** (-4 + (i % 5) * 0.5)      # layers differ in the size of their gradients
        grad = _randn(n, g) * size * used
        grad *= torch.rand(n, generator=g, device="cuda") > 0.02             # inactive units
        flat[region] = dict(p=_randn(n, g) * 0.03 * used, g=grad,
                            m=_randn(n, g) * 0.4 * size * used,
                            r=(0.5 + torch.rand(n, generator=g, device="cuda")) * size * used)
    f8, f32 = flat[8], flat[32]
    codes_m, scale_m = _quantise(f8["m"].view(-1, BLOCK))
    codes_r, scale_r = _quantise(f8["r"].view(-1, BLOCK))
    s = dict(case=case, rows=rows, p8=f8["p"], g8=f8["g"], codes_m=codes_m.view(-1), scale_m=scale_m,
             codes_r=codes_r.view(-1), scale_r=scale_r, p32=f32["p"], g32=f32["g"], m32=f32["m"],
             v32=f32["r"].square(), steps=50, lr=1e-4, eps=1e-8)
    if own:                                  # the optimizer a training program keeps, with this state loaded
        s["opt"] = _optimizer(s)
    return s


def _views(s):
    params = []
    for shape, region, a in s["rows"]:
        n = math.prod(shape)
        p = torch.nn.Parameter(s["p%d" % region][a:a + n].view(shape))
        p.grad = s["g%d" % region][a:a + n].view(shape)
        params.append(p)
    return params


def _optimizer(s):
    from unet_amd.optim import ClipAdamW
    case, params = s["case"], _views(s)
    opt = ClipAdamW(params, lr=s["lr"], betas=BETAS, eps=s["eps"], weight_decay=case["decay"],
                    max_grad_norm=case["clip"] or None, state_bits=8, min_8bit_numel=SMALL)
    state = {}
    for i, (shape, region, a) in enumerate(s["rows"]):
        n = math.prod(shape)
        b0, b1 = a // BLOCK, -(-(a + n) // BLOCK)
        step = torch.tensor(float(s["steps"]))
        if region == 8:
            state[i] = dict(step=step, exp_avg=s["codes_m"][a:a + n].view(shape), exp_avg_scale=s["scale_m"][b0:b1],
                            exp_avg_sq_root=s["codes_r"][a:a + n].view(shape), exp_avg_sq_root_scale=s["scale_r"][b0:b1])
        else:
            state[i] = dict(step=step, exp_avg=s["m32"][a:a + n].view(shape), exp_avg_sq=s["v32"][a:a + n].view(shape))
    opt.load_state_dict(dict(state=state, param_groups=opt.state_dict()["param_groups"]))
    for k in ("codes_m", "scale_m", "codes_r", "scale_r", "m32", "v32"):     # the optimizer holds its own
        del s[k]
    return opt


def prepare(case, seed):
    if case["op"] == "adam":
        return _prepare_adam(case, seed)
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    n, c = case["n"], case["c"]
    s = dict(case=case)
    if case["op"] == "scan_step":
        s.update(x=_randn((n, c), g).to(dt), gate=(_randn((n, c), g) * 2 + 1).to(dt), state=_randn((n, c), g))
        return s
    l = case["l"]
    if case["op"] == "scan":
        # gates as a trained layer has them: most channels remember for a few rows, some for thousands
        memory = torch.rand((1, 1, c), generator=g, device="cuda") * 8 - 1
        x, gate = _randn((n, l, c), g), _randn((n, l, c), g) + memory
        if case["strided"]:                  # two column ranges of one projection
            both = torch.cat([x, gate], dim=2).to(dt)
            s["x"], s["gate"] = both[:, :, :c], both[:, :, c:]
        else:
            s["x"], s["gate"] = x.to(dt), gate.to(dt)
        s["h0"] = _randn((n, c), g) if case["state"] else None
        if case["train"]:
            s["dh"] = _randn((n, l, c), g).to(dt)
            s["dlast"] = _randn((n, c), g) if case["state"] else None
        return s
    for k in ("q", "k", "v"):
        s[k] = _randn((n, l, c), g).to(dt)
    s["q"] = s["q"] * 1.5
    table = _randn((case["buckets"], case["heads"]), g)
    if case["local"]:                        # the outermost bucket of each side takes no part
        side = case["buckets"] // 2
        table[side - 1] = -math.inf
        table[2 * side - 1] = -math.inf
    s["table"] = table.to(dt)
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    s["scale"] = 1.0 / math.sqrt(c // case["heads"])
    if case["train"]:
        s["dout"] = _randn((n, l, c), g).to(dt)
    return s


# ---------------------------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"scan": _run_scan, "scan_step": _run_step, "rel": _run_rel, "adam": _run_adam}[s["case"]["op"]](s)


def _run_step(s):
    """One more row of every sequence; the carried state moves on in place."""
    if own:
        from unet_amd import ops
        return dict(h=ops.gated_scan_step(s["x"], s["gate"], s["state"]), state=s["state"])
    f = torch.sigmoid(s["gate"].float())
    s["state"].copy_(f * s["state"] + torch.sigmoid(-s["gate"].float()) * s["x"].float())
    return dict(h=s["state"].to(s["x"].dtype), state=s["state"])


def _doubling(f, b):
    """h_t = f_t h_{t-1} + b_t along dim 1, by combining spans of 1, 2, 4, ... rows."""
    d, l = 1, f.shape[1]
    f, b = f.clone(), b.clone()
    while d < l:
        b[:, d:] += f[:, d:] * b[:, :-d].clone()
        f[:, d:] *= f[:, :-d].clone()
        d *= 2
    return f, b


def _run_scan(s):
    case = s["case"]
    train, rev, dt = case["train"], case["reverse"], s["x"].dtype
    if own:
        from unet_amd import ops
        if not train:
            h, last = ops.gated_scan(s["x"], s["gate"], s["h0"], reverse=rev, return_state=True)
            return dict(h=h, last=last)
        x, gate = s["x"].detach().requires_grad_(), s["gate"].detach().requires_grad_()
        leaves = [x, gate]
        h0 = s["h0"]
        if h0 is not None:
            h0 = h0.detach().requires_grad_()
            leaves.append(h0)
        h, last = ops.gated_scan(x, gate, h0, reverse=rev, return_state=True)
        if h0 is not None:
            got = torch.autograd.grad([h, last], leaves, [s["dh"], s["dlast"]])
        else:
            got = torch.autograd.grad(h, leaves, s["dh"])
        return dict(h=h.detach(), last=last.detach(), grads=list(got))
    x, gate = s["x"].float(), s["gate"].float()
    if rev:
        x, gate = x.flip(1), gate.flip(1)
    f, fc = torch.sigmoid(gate), torch.sigmoid(-gate)
    decay, h = _doubling(f, fc * x)
    first = s["h0"] if s["h0"] is not None else torch.zeros_like(h[:, 0])
    h = h + decay * first[:, None]
    out = dict(h=(h.flip(1) if rev else h).to(dt), last=h[:, -1].clone())
    if train:
        dh = s["dh"].float()
        if rev:
            dh = dh.flip(1)
        dh = dh.clone()
        if s["dlast"] is not None:
            dh[:, -1] += s["dlast"]
        # lam_t = dh_t + f_{t+1} lam_{t+1}: the same recurrence from the other end
        fn = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], dim=1)
        lam = _doubling(fn.flip(1), dh.flip(1))[1].flip(1)
        prev = torch.cat([first[:, None], h[:, :-1]], dim=1)
        dx, dg = lam * fc, lam * (prev - x) * f * fc
        if rev:
            dx, dg = dx.flip(1), dg.flip(1)
        out["grads"] = [dx.to(dt), dg.to(dt)]
        if s["h0"] is not None:
            out["grads"].append(lam[:, 0] * f[:, 0])
    return out


def _buckets_of(case, off):
    """Bucket of key j seen from query i, off = j - i: side 0 for j <= i, side 1 for j > i."""
    starts = torch.tensor(_starts(case["buckets"], case["distance"]), device="cuda")
    b = torch.bucketize(off.abs(), starts, right=True) - 1
    return b + (off > 0) * (case["buckets"] // 2)


def _run_rel(s):
    case = s["case"]
    n, l, c, nh, dt = case["n"], case["l"], case["c"], case["heads"], s["q"].dtype
    if own:
        from unet_amd import ops
        kw = dict(n_heads=nh, scale=s["scale"], max_distance=case["distance"], lengths=s["lengths"])
        if not case["train"]:
            with torch.no_grad():
                return ops.rel_bias_attention(s["q"], s["k"], s["v"], s["table"], **kw)
        leaves = [s[k].detach().requires_grad_() for k in ("q", "k", "v", "table")]
        out = ops.rel_bias_attention(*leaves, **kw)
        return dict(out=out.detach(), grads=list(torch.autograd.grad(out, leaves, s["dout"])))
    heads = lambda t: t.float().view(n, l, nh, c // nh).transpose(1, 2).contiguous()
    flat = lambda t: t.transpose(1, 2).reshape(n, l, c).to(dt)
    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    off = torch.arange(1 - l, l, device="cuda")
    by_off = s["table"].float()[_buckets_of(case, off)].t().contiguous()     # [H, 2 L - 1]: one bias per offset j - i
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    score += by_off.unfold(1, l, 1).flip(1)                                  # row i starts at offset -i
    if s["lengths"] is not None:
        ok = torch.arange(l, device="cuda")[None, :] < s["lengths"][:, None]
        score = torch.where((ok[:, None, :] & ok[:, :, None])[:, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    prob = torch.exp(score - top)
    total = prob.sum(-1, keepdim=True)
    prob = prob / torch.where(total == 0, torch.ones_like(total), total)     # a row with nothing to see gives zeros
    out = torch.matmul(prob, v)
    if not case["train"]:
        return flat(out)
    do = heads(s["dout"])
    dv = torch.matmul(prob.transpose(2, 3).contiguous(), do)
    ds = prob * (torch.matmul(do, v.transpose(2, 3).contiguous()) - (do * out).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * s["scale"]
    pos = torch.arange(l, device="cuda")
    picks = (_buckets_of(case, pos[None, :] - pos[:, None]).reshape(-1, 1) == torch.arange(case["buckets"], device="cuda")).double()
    dtable = torch.matmul(picks.t().contiguous(), ds.sum(0, dtype=torch.float64).view(nh, l * l).t().contiguous())
    return dict(out=flat(out), grads=[flat(dq), flat(dk), flat(dv), dtable.to(dt)])


def _run_adam(s):
    if own:
        s["opt"].step()
        got = dict(s["opt"].moment_buffers(0))
        return dict(p8=s["p8"], p32=s["p32"], norm=s["opt"].total_norm(), codes_m=got["exp_avg8"],
                    scale_m=got["exp_avg8_scale"], codes_r=got["exp_avg_sq_root8"], scale_r=got["exp_avg_sq_root8_scale"],
                    m32=got["exp_avg"], v32=got["exp_avg_sq"])
    case = s["case"]
    s["steps"] += 1
    b1, b2 = BETAS
    size, root = s["lr"] / (1 - b1 ** s["steps"]), 1 / math.sqrt(1 - b2 ** s["steps"])
    keep = 1 - s["lr"] * case["decay"]
    norm = (s["g8"].double().square().sum() + s["g32"].double().square().sum()).sqrt().float()
    clip = torch.clamp(case["clip"] / (norm + 1e-6), max=1.0) if case["clip"] else torch.ones_like(norm)
    # 32-bit region
    g = s["g32"] * clip
    s["m32"].mul_(b1).add_(g * (1 - b1))
    s["v32"].mul_(b2).add_(g * (1 - b2) * g)
    s["p32"].mul_(keep).sub_(s["m32"] / (s["v32"].sqrt() * root + s["eps"]) * size)
    # 8-bit region: moments read from their codes, moved on in 32 bits, stored back
    if s["g8"].numel():
        g = (s["g8"] * clip).view(-1, BLOCK)
        m = s["codes_m"].float().view(-1, BLOCK) * s["scale_m"][:, None]
        r = s["codes_r"].float().view(-1, BLOCK) * s["scale_r"][:, None]
        m = m * b1 + g * (1 - b1)
        r = (r * r * b2 + g * (1 - b2) * g).sqrt()
        s["p8"].mul_(keep).sub_((m / (r * root + s["eps"]) * size).view(-1))
        codes, scale = _quantise(m)
        s["codes_m"].copy_(codes.view(-1)), s["scale_m"].copy_(scale)
        codes, scale = _quantise(r)
        least = torch.full_like(codes.float(), 2.0 ** -9)
        codes = torch.where((r > 0) & (codes.float() == 0), least, codes.float()).to(torch.float8_e4m3fn)
        s["codes_r"].copy_(codes.view(-1)), s["scale_r"].copy_(scale)
    return dict(p8=s["p8"], p32=s["p32"], norm=norm, codes_m=s["codes_m"], scale_m=s["scale_m"], codes_r=s["codes_r"],
                scale_r=s["scale_r"], m32=s["m32"], v32=s["v32"])


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adam":
        _, end = _layout(case)
        # p, g and both moments read; p and both moments written; one fp32 scale per block and moment each way
        return dict(bytes=end[8] * (16 + 16 / BLOCK) + end[32] * 28, flops=18 * (end[8] + end[32]))
    n, c, e = case["n"], case["c"], SIZE[case["dtype"]]
    if case["op"] == "scan_step":
        return dict(bytes=n * c * (3 * e + 8), flops=10 * n * c)
    l = case["l"]
    if case["op"] == "scan":
        vecs = (2 if case["state"] else 1) * 4 * n * c
        if not case["train"]:
            return dict(bytes=3 * n * l * c * e + vecs, flops=10 * n * l * c)
        return dict(bytes=6 * n * l * c * e + vecs + (8 * n * c if case["state"] else 0), flops=30 * n * l * c)
    pairs = sum(x * x for x in _lengths(case)) if case["ragged"] else n * l * l
    t = case["buckets"] * case["heads"] * e
    return dict(bytes=(8 if case["train"] else 4) * n * l * c * e + t * (2 if case["train"] else 1),
                flops=(14 if case["train"] else 4) * pairs * c)


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"scan": _exact_scan, "scan_step": _exact_step, "rel": _exact_rel, "adam": _exact_adam}[case["op"]](s)


def _exact_step(s):
    f = 1.0 / (1.0 + torch.exp(-s["gate"].double()))
    h = f * s["state"].double() + s["x"].double() / (1.0 + torch.exp(s["gate"].double()))
    return dict(h=h, state=h.clone())


def _exact_scan(s):
    case, x, gate = s["case"], s["x"].double(), s["gate"].double()
    l, order = case["l"], list(range(case["l"]))
    if case["reverse"]:
        order.reverse()
    f = 1.0 / (1.0 + torch.exp(-gate))
    keep = 1.0 / (1.0 + torch.exp(gate))
    h = torch.empty_like(x)
    start = torch.zeros_like(x[:, 0]) if s["h0"] is None else s["h0"].double()
    state = start
    for t in order:
        state = torch.addcmul(keep[:, t] * x[:, t], f[:, t], state, out=h[:, t])
    out = dict(h=h, last=state.clone())
    if not case["train"]:
        return out
    lam = s["dlast"].double() if s["dlast"] is not None else torch.zeros_like(start)
    dx, dg = torch.empty_like(x), torch.empty_like(x)
    for i in range(l - 1, -1, -1):
        t = order[i]
        before = h[:, order[i - 1]] if i else start
        lam = lam + s["dh"][:, t].double()                 # d loss / d h_t, all later rows included
        dx[:, t] = lam * keep[:, t]
        dg[:, t] = lam * (before - x[:, t]) * f[:, t] * keep[:, t]
        lam = lam * f[:, t]
    out["grads"] = [dx, dg] + ([lam] if s["h0"] is not None else [])
    return out


def _exact_rel(s):
    case = s["case"]
    n, l, nh = case["n"], case["l"], case["heads"]
    hd = case["c"] // nh
    side, starts = case["buckets"] // 2, _starts(case["buckets"], case["distance"])
    row = [0] * (2 * l - 1)                                  # bucket by offset j - i, from -(l - 1) to l - 1
    for off in range(-(l - 1), l):
        b = max(k for k, a in enumerate(starts) if a <= abs(off))
        row[off + l - 1] = b + (side if off > 0 else 0)
    row = torch.tensor(row, device="cuda")
    pos = torch.arange(l, device="cuda")
    idx = row[(pos[None, :] - pos[:, None]) + l - 1]
    out = torch.zeros((n, l, case["c"]), dtype=torch.float64, device="cuda")
    grads = [torch.zeros_like(out) for _ in range(3)] if case["train"] else []
    dtable = torch.zeros((case["buckets"], nh), dtype=torch.float64, device="cuda")
    lens = [l] * n if s["lengths"] is None else s["lengths"].tolist()
    for w in range(n):
        m = lens[w]
        if m == 0:
            continue
        at = idx[:m, :m]
        for hh in range(nh):
            cols = slice(hh * hd, (hh + 1) * hd)
            q, k, v = (s[x][w, :m, cols].double() for x in ("q", "k", "v"))
            z = torch.mm(q, k.t()) * s["scale"] + s["table"].double()[:, hh][at]
            p = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
            o = torch.mm(p, v)
            out[w, :m, cols] = o
            if case["train"]:
                do = s["dout"][w, :m, cols].double()
                dp = torch.mm(do, v.t())
                dz = p * (dp - (p * dp).sum(1, keepdim=True))
                grads[0][w, :m, cols] = torch.mm(dz, k) * s["scale"]
                grads[1][w, :m, cols] = torch.mm(dz.t(), q) * s["scale"]
                grads[2][w, :m, cols] = torch.mm(p.t(), do)
                # pairs of one offset lie on one diagonal: skewing the rows turns the diagonals into columns
                skew = torch.zeros((m, 2 * m), dtype=torch.float64, device="cuda")
                skew[:, :m] = dz.flip(0)
                by_off = skew.view(-1)[:m * (2 * m - 1)].view(m, 2 * m - 1).sum(0)
                dtable[:, hh].index_add_(0, row[l - m:l + m - 1], by_off)
    return dict(out=out, grads=grads + [dtable]) if case["train"] else out


def _e4m3(y):
    """Nearest e4m3 value, ties to even: three mantissa bits down to 2^-6, then steps of 2^-9."""
    mant, ex = torch.frexp(y)
    step = torch.exp2((ex - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step


def _exact_adam(s):
    case, t = s["case"], s["steps"] + 1
    b1, b2 = BETAS
    norm = math.sqrt(float((s["g8"].double() ** 2).sum()) + float((s["g32"].double() ** 2).sum()))
    clip = min(1.0, case["clip"] / (norm + 1e-6)) if case["clip"] else 1.0

    def moved(p, g, m, v):
        g = g.double() * clip
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        step = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"])
        return p.double() * (1 - s["lr"] * case["decay"]) - s["lr"] * step, m, v

    def stored(x):
        x = x.view(-1, BLOCK)
        top = x.abs().amax(1, keepdim=True)
        y = torch.where(top > 0, x / torch.where(top > 0, top, torch.ones_like(top)) * FP8_MAX, torch.zeros_like(x))
        return x, _e4m3(y), (top / FP8_MAX).squeeze(1)

    p32, m32, v32 = moved(s["p32"], s["g32"], s["m32"].double(), s["v32"].double())
    scale = lambda k: s[k].double().repeat_interleave(BLOCK)
    p8, m, v = moved(s["p8"], s["g8"], s["codes_m"].double() * scale("scale_m"),
                     (s["codes_r"].double() * scale("scale_r")) ** 2)
    _, cm, sm = stored(m)
    x, cr, sr = stored(v.sqrt())
    cr = torch.where((x > 0) & (cr == 0), torch.full_like(cr, 2.0 ** -9), cr)
    return dict(p8=p8, p32=p32, norm=torch.tensor(norm, dtype=torch.float64), codes_m=cm.view(-1), scale_m=sm,
                codes_r=cr.view(-1), scale_r=sr, m32=m32, v32=v32)
