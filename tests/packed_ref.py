"""64-bit references of the packed-note operators with ELEMENTWISE error bounds, for tests/test_gpu_packed_*.py.

Every bound counts roundings: u = 2^-24 is half a step of fp32, `step` half a step of the tensors' type (2^-24 or 2^-8,
torch.finfo(t).eps / 2).  A sum of n products in fp32 is off by at most n u times the sum of their magnitudes."""
import torch

from oracle.rng import attn_dropout_scale

U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def attn_ref(keys, values, queries, spans, cap=0.0, dout=None, keep=None, rest=True, two=False):
    """keys [R,E], values [R,F], queries [L,E] (any type, used as the numbers they hold), spans list of (start, n);
    keep: list of [L,n] dropout factors or None; rest: the backward has what the rounding of O dropped; two: P and dS enter their
    products in two pieces of the tensors' type (off by half a step of what the first one dropped).  Returns dict of name ->
    (value, bound): O, lse and, with dout [B,L,F], dK, dV, dQ."""
    step = half_step(values.dtype)
    piece = (step * step if two else step) * (step > U)
    k, v, q = (x.detach().cpu().double() for x in (keys, values, queries))
    B, L, E, F, R = len(spans), q.shape[0], k.shape[1], v.shape[1], k.shape[0]
    z = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    out = {n: [z(*s), z(*s)] for n, s in (('O', (B, L, F)), ('lse', (B, L)), ('dK', (R, E)), ('dV', (R, F)), ('dQ', (L, E)))}
    out['lse'][0].fill_(float('-inf'))
    slabs = 0
    for b, (s0, n) in enumerate(spans):
        if n == 0:
            continue
        kb, vb = k[s0:s0 + n], v[s0:s0 + n]
        x = q @ kb.T
        dx = (E + 2) * U * (q.abs() @ kb.T.abs())         # the product's sum
        if cap > 0:
            th = torch.tanh(x / cap)
            y, slope = cap * th, 1 - th * th
            dy = dx + 8 * U * cap                          # tanh from exp and reciprocal, a few roundings of values below 2
        else:
            th, y, slope, dy = None, x, 1.0, dx
        dy = dy + 4 * U * y.abs() + 4 * U                  # into units of log 2, and the exponential itself
        lse = torch.logsumexp(y, 1, keepdim=True)
        P = torch.exp(y - lse)
        dlse = (P * dy).sum(1, keepdim=True) + (n + 4) * U + 4 * U * lse.abs()
        out['lse'][0][b], out['lse'][1][b] = lse[:, 0], dlse[:, 0]
        rel = dy + dlse + 2 * U * (y - lse).abs() + 4 * U  # relative error of a weight
        D = 1.0 if keep is None else keep[b]
        Pd = P * D
        O = Pd @ vb
        dO_ = (Pd * (rel + piece + (n + 4) * U)) @ vb.abs()   # P is rounded to the tensors' type for the product
        out['O'][0][b] = O
        out['O'][1][b] = dO_ + (O.abs() + dO_) * step
        if dout is None:
            continue
        g = dout[b].detach().cpu().double()
        slabs += 1
        out['dV'][0][s0:s0 + n] = Pd.T @ g
        out['dV'][1][s0:s0 + n] = (Pd * (rel + piece + (L + 4) * U)).T @ g.abs()
        dP = g @ vb.T
        ddP = (F + 2) * U * (g.abs() @ vb.T.abs())
        delta = (g * O).sum(1, keepdim=True)
        ofO = dO_ + (O.abs() + dO_) * step * step if rest else out['O'][1][b]
        ddelta = (g.abs() * (ofO + (F + 2) * U * O.abs())).sum(1, keepdim=True)
        inner = dP * D - delta
        dS = P * inner * slope
        ddS = P * ((rel + 4 * U) * inner.abs() + ddP * D + ddelta) * (1.0 if cap == 0 else slope.abs())
        if cap > 0:
            dth = (dx / cap + 8 * U) * slope + 4 * U       # error of tanh, from x's error and its own
            ddS = ddS + P * inner.abs() * 2 * (th.abs() * dth + dth * dth + U)
        ddS = ddS + dS.abs() * piece
        out['dQ'][0] += dS @ kb
        out['dQ'][1] += (ddS + (n + 4) * U * dS.abs()) @ kb.abs()
        out['dK'][0][s0:s0 + n] = dS.T @ q
        out['dK'][1][s0:s0 + n] = (ddS + (L + 4) * U * dS.abs()).T @ q.abs()
    for name in ('dK', 'dV', 'dQ'):
        val, err = out[name]
        err += (slabs + 256) * U * err + (val.abs() + err) * step          # joining the shares; the last rounding
    return {n: tuple(x) for n, x in out.items()}


def dropout_keep(spans, L, seed, p, l_offset=0, L_total=0):
    """The counter hash's factors, as oracle/rng.py defines them, per note: [L, n]."""
    L_total = L_total or L
    return [torch.from_numpy(attn_dropout_scale(seed, [b], range(l_offset, l_offset + L), L_total, range(n), p)[0]).double()
            for b, (_, n) in enumerate(spans)]


TINY = 2.0 ** -120  # what lies below fp32's smallest normal number, 2^-126, may be flushed to zero; magnitudes it meets here: < 64


def within(got, want, what):
    val, tol = want
    tol = tol + TINY
    got = got.detach().cpu().double()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    same = (got == val) | (torch.isnan(got) & torch.isnan(val))
    bad = ~same & ~((got - val).abs() <= tol)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} outside the bound; first at {i}: got {got[tuple(i)].item()!r}, '
                             f'want {val[tuple(i)].item()!r} +- {tol[tuple(i)].item():.3e}')


def scan_ref(gates, cands, spans, h0=None, reverse=False, dh=None, dlast=None):
    """dict of name -> (value, bound): h, last and, with dh / dlast (either may be None), dg, dc, dh0.

    The state is a sum of terms (a product of gates) * (z c) or * h0.  A kernel may run through the steps or join pieces
    (A2 A1, A2 B1 + B2); either way a term passes through each of its gates once (a gate is off by a few roundings of its
    own size, and by |g| u where it is the small one of the two, from the rounded exponent) and through one addition per step or join, so its error is at most the number of its steps times 10 u, relative to
    the TERM: cancellation between terms does not shrink it.  The bound is therefore the recurrence of the terms' magnitudes,
    m_t = a_t m_{t-1} + |z_t c_t|, with e_t = a_t e_{t-1} + (10 + |g_t|) u m_t; 30 u m on top for the joins (at most 30 levels)."""
    step = half_step(gates.dtype)
    g, c = gates.detach().cpu().double(), cands.detach().cpu().double()
    R, H = g.shape
    B = len(spans)
    z = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    out = {n: [z(*s), z(*s)] for n, s in (('h', (R, H)), ('last', (B, H)), ('dg', (R, H)), ('dc', (R, H)), ('dh0', (B, H)))}
    zz, aa = torch.sigmoid(g), torch.sigmoid(-g)
    for b, (s0, n) in enumerate(spans):
        rows = list(range(s0, s0 + n))
        if reverse:
            rows.reverse()
        h = z(H) if h0 is None else h0[b].detach().cpu().double()
        e, m = z(H), h.abs()
        before, ebefore = z(R, H), z(R, H)
        for r in rows:
            before[r], ebefore[r] = h, e + 30 * U * m
            t1, t2 = aa[r] * h, zz[r] * c[r]
            coarse = 5 * U * m if step > U else 0  # (bf16 tensors: the forward takes 1 - z, off by a few u of 1)
            m = aa[r] * m + t2.abs()
            e = aa[r] * e + (10 + g[r].abs().nan_to_num(0, 0, 0)) * U * m + coarse
            h = t1 + t2
            out['h'][0][r], out['h'][1][r] = h, e + 30 * U * m + (h.abs() + e) * step
        out['last'][0][b], out['last'][1][b] = h, e + 30 * U * m
        if dh is None and dlast is None:
            continue
        carry = z(H) if dlast is None else dlast[b].detach().cpu().double()
        ec, m = z(H), carry.abs()
        for r in reversed(rows):
            up = z(H) if dh is None else dh[r].detach().cpu().double()
            lam = carry + up
            m = m + up.abs()
            el = ec + 31 * U * m
            out['dc'][0][r] = lam * zz[r]
            gr = g[r].abs().nan_to_num(0, 0, 0)
            out['dc'][1][r] = (el + (8 + gr) * U * lam.abs()) * zz[r]
            d = c[r] - before[r]
            w = zz[r] * aa[r]
            # the backward reads h as it was stored: one rounding to the tensors' type on top of its error
            ed = ebefore[r] + (before[r].abs() + ebefore[r]) * step + U * (c[r].abs() + before[r].abs())
            out['dg'][0][r] = lam * d * w
            out['dg'][1][r] = w * ((el + (20 + gr) * U * lam.abs()) * (d.abs() + ed) + lam.abs() * ed)
            m = aa[r] * m
            ec = aa[r] * ec + (10 + gr) * U * m
            carry = aa[r] * lam
        out['dh0'][0][b], out['dh0'][1][b] = carry, ec + 30 * U * m
    for name in ('dg', 'dc'):
        val, err = out[name]
        err += (val.abs() + err) * step
    return {n: tuple(x) for n, x in out.items()}
