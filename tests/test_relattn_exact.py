"""ops.rel_bias_attention in fp32 where every score is exact: small whole numbers in q and k, biases in eighths around 1000.  Then the
kernel's P has the error of exp(s - m) / l with an exact difference, 3 |s - m| u and the roundings of the sum, whatever the scores'
size; scores held in the log2 domain, or a maximum and a logarithm added up, would round at 1000 log2 e and leave 1000 times that."""
import math

import pytest
import torch

from .test_relattn import U, bucket_by_definition, call, near

N, L, HEADS, HD, BUCKETS, MAXD, SCALE = 2, 150, 2, 16, 16, 30, 0.5


def exact_inputs(dev):
    gen = torch.Generator().manual_seed(5)
    c = HEADS * HD
    q, k = (torch.randint(-1, 2, (N, L, c), generator=gen).float().to(dev) for _ in range(2))
    v, dout = (torch.randn(N, L, c, generator=gen).to(dev) for _ in range(2))
    table = 1000.0 + torch.randint(-12, 13, (BUCKETS, HEADS), generator=gen) / 8.0
    return q, k, v, table.to(dev), dout


def reference(q, k, v, table, dout):
    """float64 (value, bound) of out, dq, dk, dv, dtable, and the bound of P relative to it."""
    dev = q.device
    row = torch.tensor([bucket_by_definition(o, BUCKETS, MAXD) for o in range(1 - L, L)], device=dev)
    pos = torch.arange(L, device=dev)
    at = row[pos[None, :] - pos[:, None] + L - 1]
    val = {key: torch.zeros(N, L, HEADS * HD, dtype=torch.float64, device=dev) for key in ("out", "dq", "dk", "dv")}
    val["dtable"] = torch.zeros(BUCKETS, HEADS, dtype=torch.float64, device=dev)
    err = {key: torch.zeros_like(t) for key, t in val.items()}
    rels, scores = [], []
    for w in range(N):
        for h in range(HEADS):
            cols = slice(h * HD, (h + 1) * HD)
            Q, K, V, D = (t[w, :, cols].double() for t in (q, k, v, dout))
            S = SCALE * Q @ K.T + table[:, h].double()[at]
            below = S.amax(1, keepdim=True) - S
            P = torch.exp(-below)
            P = P / P.sum(1, keepdim=True)
            rel = U * (3 * below + 8)                              # of an exponential
            rel = rel + (rel * P).sum(1, keepdim=True) + (L + 16) * U          # .. and of their sum and its logarithm
            O = P @ V
            eO = (rel * P) @ V.abs() + L * U * (P @ V.abs()) + U * O.abs()
            dP, delta = D @ V.T, (D * O).sum(1, keepdim=True)
            edelta = (D.abs() * eO).sum(1, keepdim=True) + U * delta.abs()
            dS = P * (dP - delta)
            edS = rel * dS.abs() + P * (HD * U * (D.abs() @ V.abs().T) + edelta) + 4 * U * dS.abs()
            val["out"][w, :, cols], err["out"][w, :, cols] = O, eO
            val["dv"][w, :, cols], err["dv"][w, :, cols] = P.T @ D, ((rel + L * U) * P).T @ D.abs()
            e2 = edS + (L + 2) * U * dS.abs()
            val["dq"][w, :, cols], err["dq"][w, :, cols] = SCALE * dS @ K, SCALE * e2 @ K.abs()
            val["dk"][w, :, cols], err["dk"][w, :, cols] = SCALE * dS.T @ Q, SCALE * e2.T @ Q.abs()
            val["dtable"][:, h].index_add_(0, at.reshape(-1), dS.reshape(-1))
            err["dtable"][:, h].index_add_(0, at.reshape(-1), (edS + 256 * U * dS.abs()).reshape(-1))
            rels.append(rel)
            scores.append((S, P))
    return {key: (val[key], err[key]) for key in val}, rels, scores


def test_the_bound_tells_the_log2_domain_apart_on_cpu():
    """P from scores rounded in the log2 domain, as exp2(s log2 e - (m + log2 l)), is outside of what the next test allows."""
    _, rels, scores = reference(*exact_inputs("cpu"))
    for rel, (S, P) in zip(rels, scores):
        s2 = (S.float() * torch.tensor(math.log2(math.e)))
        m = s2.amax(1, keepdim=True)
        old = torch.exp2(s2 - (m + torch.exp2(s2 - m).sum(1, keepdim=True).log2()))
        assert float(((old.double() - P).abs() / (rel * P)).max()) > 4


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [1, 64])
def test_exact_scores(copies):
    """A launch whose waves share rows, and one that fills the chip."""
    q, k, v, table, dout = exact_inputs("cuda")
    want, _, _ = reference(q, k, v, table, dout)
    got = call(*(t.repeat(copies, 1, 1) for t in (q, k, v)), table, dout.repeat(copies, 1, 1), n_heads=HEADS, scale=SCALE, max_distance=MAXD)
    for key in ("out", "dq", "dk", "dv"):
        for w in (0, copies - 1):
            near(got[key][w * N:w * N + N], want[key], key)
    value, bound = want["dtable"]
    near(got["dtable"], (value * copies, bound * copies), "dtable")
