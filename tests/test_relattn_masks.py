"""ops.rel_bias_attention where a table's mask is a large FINITE number (-1e9, the type's lowest value): a row that sees nothing
else has equal scores, in every tile, share and pass.

Next to numbers of that size a score of a few tens vanishes (an ulp of 1e9 is 64, in the log2 domain 128), so the reference gives
such a row P = 1 / m over its m keys.  P is then off by its own roundings only, (m + 8) u; everything else is bounded as in
test_relattn.py, whose oracle covers the other rows (there a masked pair is a removed one)."""
import math

import pytest
import torch

from .test_relattn import U, bucket_by_definition, call, inputs, near, oracle

LOWEST = torch.finfo(torch.float32).min
# buckets that hold the mask, of 16 with borders up to distance 30: everything; all but the last one behind the query (the last
# rows of a window see only masked keys, far and near); all but the last one in front of it (the first rows); all in front
MASKED = dict(all=list(range(16)), far_behind_open=list(range(15)), far_front_open=[b for b in range(16) if b != 7], front=list(range(8)))


def add_equal_rows(want, q, k, v, masked, nh, maxd, lengths, dout):
    """Adds the rows that see masked pairs only to the oracle's values and bounds; returns how many there were."""
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 0.0
    fine = half * half
    n, l, c = q.shape
    hd = c // nh
    scale = hd ** -0.5
    rest, dq_rest = fine if l <= 128 else half, fine if l <= 128 or hd <= 32 else half
    row = torch.tensor([bucket_by_definition(o, masked.shape[0], maxd) for o in range(1 - l, l)], device=q.device)
    pos = torch.arange(l, device=q.device)
    idx = row[pos[None, :] - pos[:, None] + l - 1]
    val, err = ({key: want[key][i] for key in want} for i in (0, 1))
    count = 0
    for w in range(n):
        m = l if lengths is None else max(0, min(l, int(lengths[w])))
        for h in range(nh):
            R = torch.isinf(masked[:, h][idx[:m, :m]]).all(1).nonzero()[:, 0] if m else []
            if not len(R):
                continue
            count += len(R)
            cols = slice(h * hd, (h + 1) * hd)
            Q, K, V, D = (t[w, :m, cols].double() for t in (q, k, v, dout))
            Q, D = Q[R], D[R]
            P = torch.full((len(R), m), 1.0 / m, dtype=torch.float64, device=q.device)
            eP = 2 * (m + 8) * U * P
            O, mag = P @ V, P @ V.abs()
            val["infer"][w, R, cols], err["infer"][w, R, cols] = O, eP @ V.abs() + (rest + m * U) * mag
            eO = eP @ V.abs() + (fine + m * U) * mag
            val["out"][w, R, cols], err["out"][w, R, cols] = O, eO
            dP = D @ V.T
            delta = (D * O).sum(1, keepdim=True)
            edelta = (D.abs() * (eO + fine * O.abs())).sum(1, keepdim=True) + hd * U * (D.abs() * O.abs()).sum(1, keepdim=True)
            dS = P * (dP - delta)
            edS = eP * (dP - delta).abs() + P * (hd * U * (D.abs() @ V.abs().T) + edelta) + 4 * U * dS.abs()
            val["dv"][w, :m, cols] += P.T @ D
            err["dv"][w, :m, cols] += (eP + (rest + m * U) * P).T @ D.abs()
            val["dq"][w, R, cols] = scale * dS @ K
            err["dq"][w, R, cols] = scale * (edS + (dq_rest + m * U) * dS.abs()) @ K.abs()
            val["dk"][w, :m, cols] += scale * dS.T @ Q
            err["dk"][w, :m, cols] += scale * (edS + (rest + m * U) * dS.abs()).T @ Q.abs()
            at = idx[R][:, :m].reshape(-1)
            val["dtable"][:, h].index_add_(0, at, dS.reshape(-1))
            err["dtable"][:, h].index_add_(0, at, (edS + 256 * U * dS.abs()).reshape(-1))
    return count


def check(l, hd, dtype, name, fill, lengths=None):
    from unet_amd import ops
    n = 1 if lengths is None else len(lengths)
    q, k, v, table, dout = inputs(n, l, 2, hd, 16, dtype, seed=l + hd)
    q = q / 4                                               # |scores| stay far below half an ulp of the mask
    lengths = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    t, masked = table.clone(), table.clone()
    t[MASKED[name]], masked[MASKED[name]] = fill, -math.inf
    got = call(q, k, v, t, dout, n_heads=2, max_distance=30, lengths=lengths)
    with torch.no_grad():
        got["infer"] = ops.rel_bias_attention(q, k, v, t, 2, max_distance=30, lengths=lengths)
    want = oracle(q, k, v, masked, 2, hd ** -0.5, 30, lengths, dout)
    assert add_equal_rows(want, q, k, v, masked, 2, 30, lengths, dout) > 0
    for key in got:
        near(got[key], want[key], (name, fill, key, l))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", [-1e9, LOWEST])
@pytest.mark.parametrize("name", list(MASKED))
@pytest.mark.parametrize("l,hd", [(50, 32), (400, 32), (300, 72), (1600, 64), (300, 256)])
def test_rows_that_see_only_a_finite_mask(l, hd, name, fill, dtype):
    """Near and far tiles, several tiles, a window cut in shares."""
    check(l, hd, dtype, name, fill)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fill", [-1e9, LOWEST])
def test_finite_masks_in_a_padded_batch(fill, dtype):
    check(300, 32, dtype, "far_behind_open", fill, lengths=[300, 0, 129, 1])
    check(200, 32, dtype, "all", fill, lengths=[77, 200])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [1e9, torch.finfo(torch.float32).max])
@pytest.mark.parametrize("l,hd", [(100, 32), (1600, 64)])
def test_biases_of_the_highest_value(l, hd, top, dtype):
    """The other end: where two far buckets hold a bias beside which scores vanish, every row weighs the keys of those alike, as if the
    others were removed."""
    q, k, v, table, dout = inputs(1, l, 2, hd, 16, dtype, seed=l)
    q = q / 4
    t, only = table.clone(), torch.full_like(table, -math.inf)
    t[[7, 15]] = top
    got = call(q, k, v, t, dout, n_heads=2, max_distance=30)
    # equal scores: those of q = 0 and a zero bias; dk needs q, so the rows' share of it is rebuilt from dS = P (dP - delta)
    only[[7, 15]] = 0.0
    want = oracle(torch.zeros_like(q), k, v, only, 2, hd ** -0.5, 30, None, dout)
    for key in ("out", "dq", "dv", "dtable"):
        near(got[key], want[key], (key, top))
    real = oracle(q, k, v, only, 2, hd ** -0.5, 30, None, dout)["dk"][1]
    row = torch.tensor([bucket_by_definition(o, 16, 30) for o in range(1 - l, l)], device="cuda")
    pos = torch.arange(l, device="cuda")
    far = torch.isin(row[pos[None, :] - pos[:, None] + l - 1], torch.tensor([7, 15], device="cuda")).double()
    P = far / far.sum(1, keepdim=True)
    dk = torch.zeros_like(real)
    for h in range(2):
        cols = slice(h * hd, (h + 1) * hd)
        Q, V, D = (x[0, :, cols].double() for x in (q, v, dout))
        dP = D @ V.T
        dk[0, :, cols] = hd ** -0.5 * (P * (dP - (P * dP).sum(1, keepdim=True))).T @ Q
    near(got["dk"], (dk, real), ("dk", top))
