"""Attention with a learned relative-position bias (ops.rel_bias_attention): refusals and buckets on the CPU, values and
gradients on the GPU against a plain evaluation in float64.

Tolerances are first-order error bounds evaluated in float64 next to the values.  With u = 2^-24 and r = 2^-8 (bf16) or 0 (fp32):
  score:  an fp32 sum of hd products, then 3 more roundings in the log2 domain, and the stored maximum / lse of its size:
          ds = u ((hd + 4) scale |q| |k| + 8 (|S| + max_j |S| + 1)), so P is off by 2 ds relative
  P V, P^T dO, dS K, dS^T Q: operands P and dS to f relative, an fp32 sum of L terms (L u), the result rounded once; f = r^2
  (a value and the rounded rest of it) for windows of at most 128 rows, for P V where gradients follow and for dS K with heads of
  at most 32, else r
  delta = <dO, O> takes O to r^2: its error is |dO| . err(O) + hd u |dO| |O|
  dS = P (dP - delta): err = 2 ds |dS| + P (hd u |dO| |V| + err(delta)) + 4 u |dS|
  d table: sums of dS (before the rounding to bf16) in fp32, at most 64 terms deep inside a tile row, then one per tile and
  workgroup: 256 u relative to the sum of |dS|, and the rounding to the table's type."""
import math

import pytest
import torch

U = 2.0 ** -24


def bucket_by_definition(off, n_buckets, max_distance):
    """The bucket of one offset straight from the definition, in whole numbers."""
    side = n_buckets // 2
    e = side // 2
    m = side - e
    a = abs(off)
    if a < e:
        b = a
    else:
        b = e
        for k in range(1, m):
            if a ** m * e ** k >= max_distance ** k * e ** m:
                b = e + k
    return b + (side if off > 0 else 0)


def oracle(q, k, v, table, nh, scale, maxd, lengths, dout):
    """float64 (value, bound) pairs: out, dq, dk, dv, dtable."""
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    dev = q.device
    n, l, c = q.shape
    hd = c // nh
    B = table.shape[0]
    row = torch.tensor([bucket_by_definition(o, B, maxd) for o in range(1 - l, l)], device=dev)
    pos = torch.arange(l, device=dev)
    idx = row[pos[None, :] - pos[:, None] + l - 1]
    T = table.detach().double()
    z = lambda: torch.zeros((n, l, c), dtype=torch.float64, device=dev)
    fine = half * half
    rest = fine if l <= 128 else half
    val = dict(out=z(), infer=z(), dq=z(), dk=z(), dv=z(), dtable=torch.zeros((B, nh), dtype=torch.float64, device=dev))
    err = {key: torch.zeros_like(t) for key, t in val.items()}
    picks = None
    for w in range(n):
        m = l if lengths is None else max(0, min(l, int(lengths[w])))
        if m == 0:
            continue
        at = idx[:m, :m]
        for h in range(nh):
            cols = slice(h * hd, (h + 1) * hd)
            Q, K, V = (t[w, :m, cols].detach().double() for t in (q, k, v))
            S = scale * Q @ K.T + T[:, h][at]
            fin = torch.where(torch.isfinite(S), S.abs(), torch.zeros_like(S))
            mx = S.amax(1, keepdim=True)
            mx = torch.where(torch.isfinite(mx), mx, torch.zeros_like(mx))
            P = torch.exp(S - mx)
            tot = P.sum(1, keepdim=True)
            P = P / torch.where(tot == 0, torch.ones_like(tot), tot)
            ds = U * ((hd + 4) * scale * Q.abs() @ K.abs().T + 8 * (fin + fin.amax(1, keepdim=True) + 1))
            eP = P * (2 * ds + (2 * ds * P).sum(1, keepdim=True) + (m + 8) * U)
            O = P @ V
            val["infer"][w, :m, cols], err["infer"][w, :m, cols] = O, eP @ V.abs() + (rest + m * U) * (P @ V.abs())
            eO = eP @ V.abs() + (fine + m * U) * (P @ V.abs())
            val["out"][w, :m, cols], err["out"][w, :m, cols] = O, eO
            if dout is None:
                continue
            D = dout[w, :m, cols].double()
            dP = D @ V.T
            eO = eO + fine * O.abs()                       # as stored: a value and its rest
            delta = (D * O).sum(1, keepdim=True)
            edelta = (D.abs() * eO).sum(1, keepdim=True) + hd * U * (D.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (dP - delta)
            edS = eP * (dP - delta).abs() + P * (hd * U * (D.abs() @ V.abs().T) + edelta) + 4 * U * dS.abs()
            val["dv"][w, :m, cols] = P.T @ D
            err["dv"][w, :m, cols] = (eP + (rest + m * U) * P).T @ D.abs()
            e2 = edS + (rest + m * U) * dS.abs()
            val["dq"][w, :m, cols], err["dq"][w, :m, cols] = scale * dS @ K, scale * (e2 if hd > 32 else edS + (fine + m * U) * dS.abs()) @ K.abs()
            val["dk"][w, :m, cols], err["dk"][w, :m, cols] = scale * dS.T @ Q, scale * e2.T @ Q.abs()
            val["dtable"][:, h].index_add_(0, at.reshape(-1), dS.reshape(-1))
            err["dtable"][:, h].index_add_(0, at.reshape(-1), (edS + 256 * U * dS.abs()).reshape(-1))
    return {key: (val[key], err[key]) for key in val}


def near(got, want, what):
    value, bound = want
    half = torch.finfo(got.dtype).eps / 2
    got = got.detach().double()
    assert bool(torch.isfinite(got).all()), what
    # second-order terms of the bound: 2 %
    tol = 1.02 * bound + half * (value.abs() + bound) + 1e-30
    worst = float(((got - value).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} tolerances"


def inputs(n, l, nh, hd, buckets, dtype, seed=0, tdtype=torch.float32, dev="cuda"):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    c = nh * hd
    q, k, v, d = ((1.0 if i else 1.5) * r(n, l, c) for i in range(4))
    return [t.to(dtype).to(dev) for t in (q, k, v)] + [r(buckets, nh).to(tdtype).to(dev), d.to(dtype).to(dev)]


def call(q, k, v, table, dout, **kw):
    from unet_amd import ops
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    out = ops.rel_bias_attention(*leaves, **kw)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out,) + torch.autograd.grad(out, leaves, dout)))


def verify(q, k, v, table, dout, nh, maxd, lengths=None, scale=None, what=""):
    kw = dict(n_heads=nh, scale=scale, max_distance=maxd, lengths=lengths)
    got = call(q, k, v, table, dout, **kw)
    hd = q.shape[2] // nh
    want = oracle(q, k, v, table, nh, hd ** -0.5 if scale is None else scale, maxd, lengths, dout)
    for key in got:
        near(got[key], want[key], (what, key))
    return got


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("buckets,maxd", [(32, 128), (16, 50), (4, 2), (4, 512), (6, 7), (64, 17), (64, 512), (256, 300), (10, 64)])
def test_buckets_on_cpu(buckets, maxd):
    from unet_amd import ops
    off = torch.arange(-600, 601)
    want = [bucket_by_definition(int(o), buckets, maxd) for o in off]
    assert ops.rel_bucket(off, buckets, maxd).tolist() == want
    starts = ops.rel_bucket_starts(buckets, maxd)
    assert len(starts) == buckets // 2 and starts[0] == 0 and starts[-1] <= maxd and list(starts) == sorted(starts)


def test_oracle_gradients_against_autograd_on_cpu():
    q, k, v, table, dout = (t.double() for t in inputs(2, 13, 2, 4, 8, torch.float32, dev="cpu"))
    from unet_amd import ops
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    pos = torch.arange(13)
    bias = leaves[3][ops.rel_bucket(pos[None, :] - pos[:, None], 8, 5)]
    outs = []
    for h in range(2):
        cols = slice(4 * h, 4 * h + 4)
        outs.append(torch.softmax(0.5 * leaves[0][..., cols] @ leaves[1][..., cols].transpose(1, 2) + bias[..., h], -1) @ leaves[2][..., cols])
    out = torch.cat(outs, -1)
    grads = torch.autograd.grad(out, leaves, dout)
    want = oracle(q, k, v, table, 2, 0.5, 5, None, dout)
    for key, g in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        assert float((want[key][0] - g).abs().max()) < 1e-12, key


def test_refusals_on_cpu():
    from unet_amd import _lib, ops
    q, t = torch.zeros(2, 5, 16), torch.zeros(8, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.rel_bias_attention(q, q, q, t, 2, max_distance=5)
    with pytest.raises(ValueError, match="must all be"):
        ops.rel_bias_attention(q, q[:, :4], q, t, 2)
    with pytest.raises(TypeError, match="one dtype"):
        ops.rel_bias_attention(q, q.bfloat16(), q, t, 2)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        ops.rel_bias_attention(q.half(), q.half(), q.half(), t, 2)
    for heads in (0, 3, 8):
        with pytest.raises(ValueError, match="heads"):
            ops.rel_bias_attention(q, q, q, torch.zeros(8, max(heads, 1)), heads)
    with pytest.raises(ValueError, match="head size"):
        ops.rel_bias_attention(q[..., :12].bfloat16(), q[..., :12].bfloat16(), q[..., :12].bfloat16(), t[:, :1], 1)
    with pytest.raises(ValueError, match="table must be"):
        ops.rel_bias_attention(q, q, q, t, 4)
    for buckets, dist in ((7, 10), (2, 10), (258, 300), (8, 2), (8, 513)):
        with pytest.raises(ValueError, match="relative-position buckets"):
            ops.rel_bias_attention(q, q, q, torch.zeros(buckets, 2), 2, max_distance=dist)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            ops.rel_bias_attention(q, q, q, t, 2, scale=scale)
    with pytest.raises(ValueError, match="head size"):
        ops.rel_bias_attention(q[..., :0], q[..., :0], q[..., :0], t, 2)
    for lengths in (torch.zeros(2), torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="lengths"):
            ops.rel_bias_attention(q, q, q, t, 2, lengths=lengths)
    import ctypes as C
    lib = _lib.load()
    st = (C.c_int32 * 2)(0, 1)

    def fwd(dtype=1, n=1, l=4, c=8, nh=1, scale=1.0, buckets=4, starts=st, q=16, rest=None, lse=None):
        return lib.unet_rel_attn_fwd(dtype, q, q, q, 16, 1, buckets, starts, None, n, l, c, nh, scale, 16, rest, lse, None, 0, None)

    for kw, msg in ((dict(q=None), b"null"), (dict(dtype=5), b"dtype"), (dict(l=0), b"shape"), (dict(c=10), b"head_dim"), (dict(q=24), b"aligned"),
                    (dict(scale=0.0), b"scale"), (dict(scale=3e38), b"scale"), (dict(buckets=3), b"buckets"), (dict(starts=(C.c_int32 * 2)(1, 1)), b"distance 0"),
                    (dict(starts=(C.c_int32 * 2)(0, 0)), b"last bucket"), (dict(starts=(C.c_int32 * 2)(0, 600)), b"last bucket"),
                    (dict(buckets=6, starts=(C.c_int32 * 3)(0, 3, 2)), b"decrease"), (dict(l=1 << 27, c=8), b"slab"),
                    (dict(dtype=0, lse=16), b"out_rest"), (dict(dtype=0, rest=16), b"out_rest"),
                    (dict(dtype=0, lse=16, rest=24), b"aligned")):
        assert fwd(**kw) == -1 and msg in lib.unet_last_error(), (kw, lib.unet_last_error())
    assert lib.unet_rel_attn_bwd(1, 16, 16, 16, 16, 1, 4, st, None, 16, 16, 16, 16, 1, 4, 8, 1, 1.0, 16, 16, 16, 16, None, 16, None, 0, None) == -1
    assert b"partial" in lib.unet_last_error()
    assert lib.unet_rel_attn_bwd(0, 16, 16, 16, 16, 1, 4, st, None, 16, None, 16, 16, 1, 4, 8, 1, 1.0, 16, 16, 16, None, None, 16, None, 0, None) == -1
    assert b"out_rest" in lib.unet_last_error()
    # few rows of a long window: shares of the keys need their workspace
    need = lib.unet_rel_attn_workspace_bytes(0, 1, 4096, 8, 1, 0)
    assert need > 0 and lib.unet_rel_attn_workspace_bytes(1, 1, 4096, 8, 1, 0) == 0
    assert fwd(dtype=0, l=4096) == -1 and b"workspace" in lib.unet_last_error()
    assert lib.unet_rel_attn_bwd(0, 16, 16, 16, 16, 1, 4, st, None, 16, 16, 16, 16, 1, 4096, 8, 1, 1.0, 16, 16, 16, None, None, 16, 16, 8,
                                 None) == -1
    assert b"workspace" in lib.unet_last_error()


# ------------------------------------------------------------------------------------------------ GPU
CASES = [  # n, l, heads, hd, buckets, max distance
    (1, 1, 1, 8, 4, 2), (2, 2, 2, 16, 8, 5), (1, 31, 3, 24, 16, 30), (2, 64, 1, 32, 32, 128), (1, 65, 2, 40, 32, 20), (3, 129, 4, 64, 32, 64),
    (1, 300, 8, 64, 32, 128), (2, 257, 2, 72, 10, 200), (1, 200, 1, 128, 64, 512), (2, 140, 2, 136, 16, 33), (1, 193, 1, 256, 256, 400),
    (1, 1000, 2, 32, 32, 90)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,l,nh,hd,buckets,maxd", CASES)
def test_values_and_gradients(n, l, nh, hd, buckets, maxd, dtype):
    q, k, v, table, dout = inputs(n, l, nh, hd, buckets, dtype, seed=l)
    verify(q, k, v, table, dout, nh, maxd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [4, 12, 20, 100, 252])
def test_fp32_head_sizes(hd):
    q, k, v, table, dout = inputs(2, 70, 2, hd, 8, torch.float32, seed=hd)
    verify(q, k, v, table, dout, 2, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_most_heads_and_channels(dtype):
    q, k, v, table, dout = inputs(1, 33, 256, 64, 16, dtype, seed=24)
    verify(q, k, v, table, dout, 256, 60)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [16, 40, 128, 256])
def test_fp32_launches_that_fill_the_chip(hd):
    """256 workgroups of 64 rows: the waves own different rows (in small launches they share them)."""
    q, k, v, table, dout = inputs(4, 200, 16, hd, 16, torch.float32, seed=hd)
    verify(q, k, v, table, dout, 16, 60, lengths=torch.tensor([200, 0, 129, 64], dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [8, 64, 128, 256])
@pytest.mark.parametrize("case", ["plain", "padded", "left", "band"])
def test_few_rows_of_a_long_window(hd, case):
    """The walked axis is cut in shares: shares behind a window's length, outside the band, with and without gradients."""
    from unet_amd import ops
    l, n = 1579, 3 if case == "padded" else 1
    q, k, v, table, dout = inputs(n, l, 2, hd, 16, torch.bfloat16, seed=hd + n)
    lengths = torch.tensor([l, 600, 0], dtype=torch.int32, device="cuda") if case == "padded" else None
    if case in ("left", "band"):
        table[15] = -math.inf                      # nothing far behind the query ..
    if case == "band":
        table[7] = -math.inf                       # .. nor far in front of it
    got = verify(q, k, v, table, dout, 2, 50, lengths=lengths, what=case)
    again = call(q, k, v, table, dout, n_heads=2, max_distance=50, lengths=lengths)
    assert all(torch.equal(got[key], again[key]) for key in got)
    near(ops.rel_bias_attention(q, k, v, table, 2, max_distance=50, lengths=lengths),
         oracle(q, k, v, table, 2, hd ** -0.5, 50, lengths, None)["infer"], "no gradients")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("l,lens", [(130, (0, 1, 64, 65, 130, 200, -3)), (300, (0, 129, 300, 256, 1, 40, 299))])
def test_padded_batches(l, lens, dtype):
    """Windows of 0 .. L valid positions; what lies behind them is NaN and reaches nothing."""
    n = len(lens)
    q, k, v, table, dout = inputs(n, l, 2, 32, 16, dtype, seed=9)
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for w, m in enumerate(lens):
        for t in (q, k, v, dout):
            t[w, max(m, 0):] = float("nan")
    clean = [torch.nan_to_num(t) for t in (q, k, v, dout)]
    got = call(q, k, v, table, dout, n_heads=2, max_distance=40, lengths=lengths)
    want = oracle(*clean[:3], table, 2, 32 ** -0.5, 40, lengths, clean[3])
    for key in got:
        near(got[key], want[key], key)
    for w, m in enumerate(lens):
        for key in ("out", "dq", "dk", "dv"):
            assert float(got[key][w, max(m, 0):].detach().float().abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_in_the_table(dtype):
    """-inf entries: local bands (both sides, one side), a causal table, a table that leaves every row, or one head, empty; and the
    type's lowest value in their place."""
    low = torch.finfo(torch.float32).min
    for l in (50, 400):
        q, k, v, table, dout = inputs(2, l, 2, 32, 16, dtype, seed=11)
        ninf = float("-inf")
        sides = dict(band=[7, 15], left=[7], right=[15], causal=list(range(8, 16)), anticausal=list(range(0, 8)), near=[0, 1, 8, 9])
        for name, rows in sides.items():
            for fill in (ninf, low):
                t = table.clone()
                t[rows] = fill
                if fill == low and name == "anticausal":
                    continue      # the last row sees only the lowest value: uniform there, tested below
                got = call(q, k, v, t, dout, n_heads=2, max_distance=30)
                masked = t.clone()
                masked[rows] = ninf
                want = oracle(q, k, v, masked, 2, 32 ** -0.5, 30, None, dout)
                for key in got:
                    near(got[key], want[key], (name, fill, key, l))
                assert float(got["dtable"][rows].abs().sum()) == 0
        t = table.clone()
        t[:, 1] = ninf
        got = verify(q, k, v, t, dout, 2, 30, what="one head empty")
        assert float(got["out"][..., 32:].float().abs().sum()) == 0 and float(got["dq"][..., 32:].float().abs().sum()) == 0
        assert float(got["dtable"][:, 1].abs().sum()) == 0
        # every entry the lowest value: a constant bias, so the softmax is over equal scores or over q k^T, never NaN
        out = call(q, k, v, torch.full_like(table, low), dout, n_heads=2, max_distance=30)
        assert all(bool(torch.isfinite(g).all()) for g in out.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores_and_biases(dtype):
    """Scores far above the first tile's maximum (the forward kernel's second walk), and biases of +-1e4."""
    q, k, v, table, dout = inputs(1, 400, 2, 32, 16, dtype, seed=13)
    k[:, 250:] *= 30
    verify(q, k, v, table, dout, 2, 30, scale=1.0, what="late maximum")
    t = table.clone()
    t[3], t[12] = 1e4, -1e4
    verify(q, k, v, t, dout, 2, 30, what="large biases")
    q[0, 7, 3] = float("nan")
    from unet_amd import ops
    out = ops.rel_bias_attention(q, k, v, table, 2, max_distance=30)
    bad = torch.isnan(out).any(-1)
    assert bool(bad[0, 7]) and int(bad.sum()) == 1


@pytest.mark.gpu
def test_zero_table_is_plain_attention_and_a_constant_changes_nothing():
    from unet_amd import ops
    q, k, v, table, dout = inputs(2, 200, 2, 64, 32, torch.bfloat16, seed=14)
    one = torch.ones((1, 1), device="cuda")
    plain = ops.cfc_attention(q[None], k[None], v[None], one, 2, 0.125)
    for t in (torch.zeros_like(table), torch.full_like(table, 2.5)):
        out = ops.rel_bias_attention(q, k, v, t, 2, scale=0.125)
        want = oracle(q, k, v, t, 2, 0.125, 128, None, None)
        near(out, want["infer"], "constant")
        near(plain, want["infer"], "band-pair kernel")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bf16_table_partial_gradients_layouts(dtype):
    from unet_amd import ops
    q, k, v, table, dout = inputs(2, 150, 2, 32, 16, dtype, seed=15, tdtype=torch.bfloat16)
    got = verify(q, k, v, table, dout, 2, 40, what="bf16 table")
    assert got["dtable"].dtype == torch.bfloat16
    # gradients for q alone, for the table alone; transposed and sliced inputs; an expanded upstream gradient
    want = oracle(q, k, v, table, 2, 32 ** -0.5, 40, None, dout)
    qr = q.clone().requires_grad_()
    (dq,) = torch.autograd.grad(ops.rel_bias_attention(qr, k, v, table, 2, max_distance=40), qr, dout)
    near(dq, want["dq"], "q alone")
    tr = table.clone().requires_grad_()
    (dt,) = torch.autograd.grad(ops.rel_bias_attention(q, k, v, tr, 2, max_distance=40), tr, dout)
    near(dt, want["dtable"], "table alone")
    both = torch.cat([q, k, v], 2).transpose(0, 1).contiguous().transpose(0, 1)
    assert not both[..., :64].is_contiguous()
    near(ops.rel_bias_attention(both[..., :64], both[..., 64:128], both[..., 128:], table, 2, max_distance=40), want["infer"], "slices")
    ones = torch.ones(1, 1, 64, dtype=dtype, device="cuda").expand(2, 150, 64)
    got = call(q, k, v, table, ones, n_heads=2, max_distance=40)
    want = oracle(q, k, v, table, 2, 32 ** -0.5, 40, None, ones)
    for key in got:
        near(got[key], want[key], (key, "expanded"))
    # q, k and v the same tensor: the three gradients add up
    x = q.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.rel_bias_attention(x, x, x, table, 2, max_distance=40), x, dout)
    w = oracle(q, q, q, table, 2, 32 ** -0.5, 40, None, dout)
    half = torch.finfo(dtype).eps / 2
    value = w["dq"][0] + w["dk"][0] + w["dv"][0]
    tol = sum(1.02 * w[t][1] + 3 * half * (w[t][0].abs() + w[t][1]) for t in ("dq", "dk", "dv")) + half * value.abs()
    assert bool(((dx.double() - value).abs() <= tol).all())
    assert ops.rel_bias_attention(q[:, :0], k[:, :0], v[:, :0], table, 2, max_distance=40).shape == (2, 0, 64)


@pytest.mark.gpu
def test_directional_differences():
    from unet_amd import ops
    q, k, v, table, dout = inputs(1, 90, 2, 16, 16, torch.float32, seed=16)
    got = call(q, k, v, table, dout, n_heads=2, max_distance=40)
    dirs = [torch.randn_like(t) for t in (q, k, v, table)]
    eps = 2.0 ** -8

    def loss(sign):
        out = ops.rel_bias_attention(*(t + sign * eps * d for t, d in zip((q, k, v, table), dirs)), 2, max_distance=40)
        return float((out.double() * dout.double()).sum())

    want = sum(float((got[key].double() * d.double()).sum()) for key, d in zip(("dq", "dk", "dv", "dtable"), dirs))
    quotient = (loss(1) - loss(-1)) / (2 * eps)
    # remainder eps^2 / 6 times a third derivative of up to a hundred per output, rounding 1e-6 / eps, over 2880 outputs
    assert abs(quotient - want) <= (20 * eps ** 2 + 1e-6 / eps) * float(dout.abs().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_bits_side_stream_and_graph_replays(dtype):
    from unet_amd import ops
    lens = torch.tensor([200, 77], dtype=torch.int32, device="cuda")
    q, k, v, table, dout = inputs(2, 200, 2, 32, 16, dtype, seed=17)
    kw = dict(n_heads=2, max_distance=40, lengths=lens)
    first = call(q, k, v, table, dout, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call(q, k, v, table, dout, **kw)
    side.synchronize()
    for key in first:
        assert torch.equal(first[key], second[key]), key
    del first, second
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rel_bias_attention(*leaves, **kw)
        grads = torch.autograd.grad(out, leaves, dout)
    for rep in range(4):
        fresh = inputs(2, 200, 2, 32, 16, dtype, seed=30 + rep)
        with torch.no_grad():
            for a, b in zip(leaves, fresh):
                a.copy_(b)
            lens.copy_(torch.tensor([200 - 50 * rep, 60 * rep], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = call(*fresh[:4], dout, **kw)
        for a, key in zip((out,) + grads, ("out", "dq", "dk", "dv", "dtable")):
            assert torch.equal(a, want[key]), (rep, key)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_flat_buffers(dtype):
    """Contiguous tensors that start off a 16-byte boundary, the upstream gradient among them."""
    from unet_amd import ops
    q, k, v, table, dout = inputs(1, 70, 2, 16, 16, dtype, seed=21)
    odd = [torch.cat([t.new_zeros(i + 1), t.reshape(-1)])[i + 1:].view(t.shape) for i, t in enumerate((q, k, v))]
    assert all(t.data_ptr() % 16 and t.is_contiguous() for t in odd)
    leaves = [t.requires_grad_() for t in odd] + [table.requires_grad_()]
    out = ops.rel_bias_attention(*leaves, n_heads=2, max_distance=40)
    flat = torch.cat([out.new_zeros(3), out.reshape(-1)])
    grads = torch.autograd.grad(flat, leaves, torch.cat([dout.new_ones(3), dout.reshape(-1)]))
    want = oracle(q, k, v, table, 2, 16 ** -0.5, 40, None, dout)
    for key, t in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        near(t, want[key], key)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    from unet_amd import ops
    q, k, v, table, dout = inputs(1, 40, 2, 16, 16, torch.bfloat16, seed=22)
    q.requires_grad_()
    out = ops.rel_bias_attention(q, k, v, table, 2)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out, q, dout, create_graph=True)


@pytest.mark.gpu
def test_slabs_just_below_two_gib():
    """[131071, 8192] bf16: byte offsets up to 2^31; a local band, so that rows at the end have an oracle of their own."""
    from unet_amd import ops
    l, nh, hd = 131071, 32, 256
    gen = torch.Generator(device="cuda").manual_seed(23)
    q, k, v, dout = (torch.randn(1, l, nh * hd, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    table = torch.randn(8, nh, generator=gen, device="cuda")
    table[3] = table[7] = -math.inf                                    # nothing at distance 4 and beyond
    got = call(q, k, v, table, dout, n_heads=nh, max_distance=4)
    del got["dtable"]
    cols, rows = slice(-hd, None), slice(l - 300, None)
    part = [t[:, rows, cols].contiguous() for t in (q, k, v)]
    want = oracle(*part, table[:, -1:], 1, hd ** -0.5, 4, None, dout[:, rows, cols].contiguous())
    for key in got:
        value, bound = want[key]
        near(got[key][:, rows, cols][:, 10:], (value[:, 10:], bound[:, 10:]), key)
    first = oracle(*(t[:, :300, :hd].contiguous() for t in (q, k, v)), table[:, :1], 1, hd ** -0.5, 4, None, dout[:, :300, :hd].contiguous())
    for key in got:
        value, bound = first[key]
        near(got[key][:, :290, :hd], (value[:, :290], bound[:, :290]), key)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("l", [300, 1600])
def test_scores_that_grow_along_the_window(hd, l):
    """Keys whose scores rise by hundreds behind the first tile, in some rows only, and rows that see nothing for many tiles: the
    running reference has to move, also inside a share of the keys."""
    q, k, v, table, dout = inputs(1, l, 2, hd, 16, torch.bfloat16, seed=hd + l)
    ramp = torch.linspace(0, 1, l, device="cuda")[None, :, None]
    k = (k * (0.1 + 12 * ramp)).to(k.dtype)
    q = q.clone()
    q[:, ::3] *= 4
    verify(q, k, v, table, dout, 2, 50, what="growing")
    table[:8] = -math.inf                          # only keys behind the query: the last rows see nothing in front of them
    verify(q, k, v, table, dout, 2, 50, what="growing, keys behind")


@pytest.mark.gpu
def test_shared_axis_in_two_graphs_at_once():
    """Windows long enough to be cut in shares: forward and backward captured twice, replayed in turn and on two streams."""
    from unet_amd import ops
    sets, graphs, outs = [], [], []
    for i in range(2):
        q, k, v, table, dout = inputs(1, 1600 + 70 * i, 2, 32, 16, torch.bfloat16, seed=31 + i)
        leaves = [t.requires_grad_() for t in (q, k, v, table)]
        sets.append((leaves, dout))
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.rel_bias_attention(*leaves, 2, max_distance=40), leaves, dout)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.rel_bias_attention(*leaves, 2, max_distance=40)
            outs.append((out.detach(),) + torch.autograd.grad(out, leaves, dout))
            del out
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        with torch.no_grad():
            for leaves, _ in sets:
                leaves[0].mul_(0.9)
                leaves[3].add_(0.1)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            if rep % 2:
                with torch.cuda.stream(s):
                    graph.replay()
            else:
                graph.replay()
        torch.cuda.synchronize()
        for (leaves, dout), got in zip(sets, outs):
            out = ops.rel_bias_attention(*leaves, 2, max_distance=40)
            want = (out.detach(),) + torch.autograd.grad(out, leaves, dout)
            del out
            assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
