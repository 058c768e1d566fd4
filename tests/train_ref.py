"""64-bit references of the training operators and the error bounds their tests use.

Bounds follow the arithmetic.  U[t] is the relative error of one rounding to type t (half a step); F32 = 2^-24 that of a 32-bit operation.  A sum of n terms held
in 32 bits is off by at most n F32 times the sum of magnitudes, so a bound is a product of magnitudes in 64 bits times such a factor.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32 = 2.0 ** -24


def within(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() - bound)
    assert not torch.isnan(off).any(), f"{what}: NaN where the reference has a value (or the reverse)"
    assert off.numel() == 0 or off.max() <= 1e-37, f"{what}: {off.max():.3g} over its bound (bound there {bound.flatten()[off.argmax()]:.3g})"


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------------------
# A lane adds up to 32 entries, 6 exchanges join a wave, up to 8 waves are joined: at most 46 additions in a row's sum.
DEPTH = 46


def layer_norm(x, w, b, eps, out_dtype):
    x = x.double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double().cpu()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    y = d * rstd * w + b
    # d = (x - m0) - c: two roundings of d, and the error of the mean of the once-centred entries
    ed = F32 * (3 * d.abs() + 2 * DEPTH * d.abs().mean(-1, keepdim=True)) + DEPTH * F32 ** 2 * DEPTH * x.abs().mean(-1, keepdim=True)
    er = (2 * DEPTH + 8) * F32                       # relative: the sum of squares (with d's error in them) under a root, the division
    e2 = (ed * d.abs()).mean(-1, keepdim=True) * rstd ** 2
    by = (ed * rstd + (d * rstd).abs() * (er + e2)) * w.abs() + 3 * F32 * ((d * rstd * w).abs() + b.abs()) + U[out_dtype] * y.abs()
    bm = F32 * (2 * mean.abs() + 2 * DEPTH * d.abs().mean(-1, keepdim=True)) + DEPTH * F32 ** 2 * DEPTH * x.abs().mean(-1, keepdim=True)
    return (y, by * 1.01), (mean.squeeze(-1), bm.squeeze(-1)), (rstd.squeeze(-1), (rstd * (er + e2)).squeeze(-1))


def layer_norm_backward(dy, x, w, eps, dtype, wtype):
    x, dy = x.double().cpu(), dy.double().cpu()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / (d.square().mean(-1, keepdim=True) + eps).sqrt()
    xh, g = d * rstd, dy * w
    a, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - a - xh * c)
    ma, mc = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    e2 = 3 * DEPTH * F32                             # relative error of xh: rstd's, and d's in units of |d| + mean |d|
    exh = e2 * (xh.abs() + xh.abs().mean(-1, keepdim=True))
    ec = (exh * g.abs()).mean(-1, keepdim=True) + 2 * DEPTH * F32 * mc
    bdx = rstd * (4 * F32 * (g.abs() + a.abs() + (xh * c).abs()) + 2 * DEPTH * F32 * ma + exh * c.abs() + xh.abs() * ec) + e2 * dx.abs() + U[dtype] * dx.abs()
    rows = (x.numel() // x.shape[-1])
    dyr, xhr, er = (t.reshape(-1, x.shape[-1]) for t in (dy, xh, exh.expand_as(xh)))
    n = (min(rows, 2048) + rows / 512 + 80) * F32    # additions on one column's way: a group's rows, the workgroup's groups, the partial rows
    dw, db = (dyr * xhr).sum(0), dyr.sum(0)
    bdw = n * (dyr * xhr).abs().sum(0) + (dyr.abs() * er).sum(0) + U[wtype] * dw.abs()
    return (dx, bdx * 1.01), (dw, bdw * 1.01), (db, n * dyr.abs().sum(0) + U[wtype] * db.abs() * 1.01)


# ---- attention -------------------------------------------------------------------------------------------------------------------------------------
def attention(q, k, v, q_ptr, k_ptr, bias=None, causal=False, scale=None, dout=None):
    """Per complex and head: (out, bound), (m, bound), (l, bound) or, with dout, (dq, dk, dv, dbias) with their bounds."""
    dtype, u = q.dtype, U[q.dtype]
    p_round = 0.0 if dtype == torch.float32 else u            # probabilities and ds are rounded to bf16 for the matrix units
    q, k, v = (t.double().cpu() for t in (q, k, v))
    bias = bias.double().cpu() if bias is not None else None
    dout = dout.double().cpu() if dout is not None else None
    H, D = q.shape[1:]
    G = H // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, bout = torch.zeros_like(q), torch.zeros_like(q)
    m, l = torch.full((H, q.shape[0]), -math.inf, dtype=torch.float64), torch.zeros(H, q.shape[0], dtype=torch.float64)
    bm, bl = torch.zeros_like(l), torch.zeros_like(l)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    bq, bk, bv = (torch.zeros_like(t) for t in (q, k, v))
    db, bb = (torch.zeros_like(bias), torch.zeros_like(bias)) if bias is not None else (None, None)
    pair = 0
    for b in range(len(q_ptr) - 1):
        i0, i1, j0, j1 = q_ptr[b], q_ptr[b + 1], k_ptr[b], k_ptr[b + 1]
        nq, nk = i1 - i0, j1 - j0
        p0, pair = pair, pair + nq * nk
        if nq == 0 or nk == 0:
            continue
        for h in range(H):
            Q, K, V = q[i0:i1, h], k[j0:j1, h // G], v[j0:j1, h // G]
            s = scale * (Q @ K.T)
            es = F32 * ((D + 2) * scale * (Q.abs() @ K.abs().T))            # a score: D products, the scale
            if bias is not None:
                B = bias[h, p0:pair].view(nq, nk)
                s = torch.where(B == -math.inf, -math.inf, s + B)
                es = es + F32 * torch.where(torch.isinf(s), 0.0, s).abs()
            if causal:
                s = torch.where(torch.ones(nq, nk, dtype=torch.bool).tril(nk - nq), s, -math.inf)
            top = s.amax(1, keepdim=True)
            base = torch.where(top == -math.inf, 0.0, top)
            e = torch.where(s == -math.inf, 0.0, torch.exp(s - base))
            # relative error of exp(s - m): both scores' errors, the difference's and the exponent's roundings
            big = torch.where(s == -math.inf, 0.0, s - base).abs()
            worst = torch.where(s == -math.inf, 0.0, es).amax(1, keepdim=True)
            rel = es + worst + F32 * (4 * big + 8)
            tot = e.sum(1, keepdim=True)
            etot = (e * rel).sum(1, keepdim=True) + (nk + 4) * F32 * tot
            div = torch.where(tot == 0, 1.0, tot)
            P = e / div
            # ... and an exponential below 2^-126, the smallest normal 32-bit number, is 0: an absolute error of up to that (over tot >= 1)
            eP = P * (rel + etot / div + 8 * F32) + torch.where(s == -math.inf, 0.0, 2.0 ** -126)
            o = P @ V
            if dout is None:
                out[i0:i1, h], m[h, i0:i1], l[h, i0:i1] = o, top[:, 0], tot[:, 0]
                bout[i0:i1, h] = (eP + (p_round + (2 * nk + 8) * F32) * P) @ V.abs() + u * o.abs()
                bm[h, i0:i1], bl[h, i0:i1] = worst[:, 0], etot[:, 0]
                continue
            dO = dout[i0:i1, h]
            dp, A = dO @ V.T, dO.abs() @ V.abs().T
            delta = (dO * o).sum(1, keepdim=True)
            # the stored out carries its own error; delta is a sum of D terms
            eo = (eP + (p_round + (2 * nk + 8) * F32) * P) @ V.abs() + u * o.abs()
            ed = (dO.abs() * eo).sum(1, keepdim=True) + (D + 2) * F32 * (dO.abs() * (o.abs() + eo)).sum(1, keepdim=True)
            ds = P * (dp - delta)
            eds = eP * (dp - delta).abs() + (P + eP) * ((D + 4) * F32 * A + ed + 4 * F32 * (dp.abs() + delta.abs()))
            eall = eds + p_round * (ds.abs() + eds)
            add = (2 * max(nk, nq * G) + 8) * F32
            dq[i0:i1, h] = scale * (ds @ K)
            bq[i0:i1, h] = scale * ((eall + add * ds.abs()) @ K.abs())
            dk[j0:j1, h // G] += scale * (ds.T @ Q)
            bk[j0:j1, h // G] += scale * ((eall + add * ds.abs()).T @ Q.abs())
            dv[j0:j1, h // G] += P.T @ dO
            bv[j0:j1, h // G] += (eP + (p_round + add) * P).T @ dO.abs()
            if bias is not None:
                db[h, p0:pair], bb[h, p0:pair] = ds.reshape(-1), eds.reshape(-1)
    if dout is None:
        return (out, bout), (m, bm), (l, bl)
    out = [(dq, bq + u * (dq.abs() + bq)), (dk, bk + u * (dk.abs() + bk)), (dv, bv + u * (dv.abs() + bv))]
    return out + [(db, bb + u * (db.abs() + bb)) if bias is not None else None]


# ---- AdamW -----------------------------------------------------------------------------------------------------------------------------------------
BLOCK = 256


def decode(code, scale, power):
    c = code.double().view(-1, BLOCK)
    x = c * c.abs() / 127.0 ** 2 if power == 2 else (c / 255.0) ** 4
    return (x * scale.double()[:, None]).view(-1)


def encode(x, power):
    """Nearest codes by comparison with the borders between neighbours."""
    top = 127 if power == 2 else 255
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1).float()
    border = ((torch.arange(top, dtype=torch.float64) + 0.5) / top) ** power
    share = torch.where(scale[:, None] > 0, x.abs() / scale.double()[:, None], torch.zeros_like(x))
    c = torch.bucketize(share, border, right=True)
    if power == 4:
        c = torch.where((share > 0) & (c == 0), 1, c)
    return (c * torch.sign(x).long()).view(-1).to(torch.int8 if power == 2 else torch.uint8), scale


def adamw(p, g, m, v, t, lr, b1, b2, eps, wd, scale=1.0):
    """(p, m, v) after step number t, and the bound of each in 32-bit arithmetic."""
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    g = g * scale
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    upd = lr * (m1 / (1 - b1 ** t)) / ((v1 / (1 - b2 ** t)).sqrt() + eps)
    p1 = p * (1 - lr * wd) - upd
    em = 4 * F32 * (b1 * m.abs() + (1 - b1) * g.abs())
    ev = 6 * F32 * v1
    # the step's relative error: m's, half of v's, and about ten roundings of factors, root and quotient
    eu = 16 * F32 * upd.abs() + lr / (1 - b1 ** t) * em / ((v1 / (1 - b2 ** t)).sqrt() + eps)
    return (p1, eu + 4 * F32 * (p.abs() + upd.abs())), (m1, em), (v1, ev + 1e-44)
