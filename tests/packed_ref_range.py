"""The 64-bit reference of the packed attention for caps of any size and for keys, queries and values of any value, infinities
among them, with elementwise bounds: tests/packed_ref.py's, but for a score's error, which here is relative to the score.

y = cap tanh(x / cap) is off by the product's own error (a sum of E products in fp32) and by at most 24 u |y|: below |x / cap| = 0.35
from an odd series of eight roundings, above it from 1 - 2 / (1 + e^{2 x / cap}), whose 8 u cap are below 24 u |y| there
(tanh(0.35) = 0.336).  A score that saturates is +-cap, off by the 8 u cap alone, whatever the product's error."""
import torch

from tests.packed_ref import U, half_step


def attn_ref_range(keys, values, queries, spans, cap=0.0, dout=None, keep=None):
    step = half_step(values.dtype)
    piece = step * step if step > U else 0.0
    k, v, q = (x.detach().cpu().double() for x in (keys, values, queries))
    B, L, E, F, R = len(spans), q.shape[0], k.shape[1], v.shape[1], k.shape[0]
    z = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    out = {n: [z(*s), z(*s)] for n, s in (('O', (B, L, F)), ('lse', (B, L)), ('dK', (R, E)), ('dV', (R, F)), ('dQ', (L, E)))}
    out['lse'][0].fill_(float('-inf'))
    for b, (s0, n) in enumerate(spans):
        if n == 0:
            continue
        kb, vb = k[s0:s0 + n], v[s0:s0 + n]
        x = q @ kb.T
        dx = (E + 2) * U * (q.abs() @ kb.T.abs())
        if cap > 0:
            th = torch.tanh(x / cap)
            y, slope = cap * th, 1 - th * th
            flat = (x / cap).abs() >= 30                     # (slope below 1e-25)
            dy = torch.where(flat, 8 * U * cap, dx + 24 * U * y.abs())
        else:
            th, y, slope = None, x, torch.ones_like(x)
            dy = torch.where(x.isinf(), 0.0, dx)
        dy = dy + torch.where(y.isinf(), 0.0, 4 * U * y.abs()) + 4 * U
        lse = torch.logsumexp(y, 1, keepdim=True)
        P = torch.exp(y - lse)
        dlse = (P * dy).sum(1, keepdim=True) + (n + 4) * U + 4 * U * lse.abs()
        out['lse'][0][b], out['lse'][1][b] = lse[:, 0], dlse[:, 0]
        rel = dy + dlse + torch.where(y.isinf(), 0.0, 2 * U * (y - lse).abs()) + 4 * U
        D = 1.0 if keep is None else keep[b]
        Pd = P * D
        O = Pd @ vb
        dO_ = (Pd * (rel + piece + (n + 4) * U)) @ vb.abs()
        out['O'][0][b] = O
        out['O'][1][b] = dO_ + (O.abs() + dO_) * step
        if dout is None:
            continue
        g = dout[b].detach().cpu().double()
        out['dV'][0][s0:s0 + n] = Pd.T @ g
        out['dV'][1][s0:s0 + n] = (Pd * (rel + piece + (L + 4) * U)).T @ g.abs()
        dP = g @ vb.T
        ddP = (F + 2) * U * (g.abs() @ vb.T.abs())
        delta = (g * O).sum(1, keepdim=True)
        ofO = dO_ + (O.abs() + dO_) * step * step
        ddelta = (g.abs() * (ofO + (F + 2) * U * O.abs())).sum(1, keepdim=True)
        inner = dP * D - delta
        dS = P * inner * slope
        ddS = P * ((rel + 4 * U) * inner.abs() + ddP * D + ddelta) * slope
        if cap > 0:
            dth = torch.where(flat, 4 * U, (dx / cap + 24 * U * th.abs()) * slope + 8 * U * th.abs())
            ddS = ddS + P * inner.abs() * 2 * (th.abs() * dth + dth * dth + U)
        ddS = ddS + dS.abs() * piece
        out['dQ'][0] += dS @ kb
        out['dQ'][1] += (ddS + (n + 4) * U * dS.abs()) @ kb.abs()
        out['dK'][0][s0:s0 + n] = dS.T @ q
        out['dK'][1][s0:s0 + n] = (ddS + (L + 4) * U * dS.abs()).T @ q.abs()
    for name in ('dK', 'dV', 'dQ'):
        val, err = out[name]
        err += (B + 256) * U * err + (val.abs() + err) * step
    return {n: tuple(x) for n, x in out.items()}
