"""The packed-note operators in one run, as a model uses them: a gated recurrence over the word vectors, label attention over its
states, per-label scores and loss, backward through all of it, and a clipped AdamW step; and the recurrence's serving form."""
import math

import pytest
import torch

from tests.packed_ref import U, attn_ref, scan_ref, within

pytestmark = pytest.mark.gpu
DEV = 'cuda'
LENS, VOCAB, H, L, CAP = [37, 0, 130, 1, 64], 50, 40, 23, 20.0


@pytest.fixture(scope='module')
def ops():
    from gzsl_text_amd.ops_hip import HipOps
    return HipOps()


@pytest.fixture(scope='module')
def ext():
    from gzsl_text_amd import torch_ext
    torch_ext.build()
    torch_ext.load()
    return torch.ops.gzsl


class Scorer(torch.nn.Module):
    """Notes -> [B, L] scores: word vectors, a gate and a candidate per channel, the recurrence, attention of every label."""

    def __init__(self, ext, seed):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        par = lambda *s: torch.nn.Parameter((0.3 * torch.randn(*s, generator=gen)).to(DEV))  # noqa: E731
        self.words, self.gate, self.cand, self.key, self.query, self.label = par(VOCAB, H), par(H, H), par(H, H), par(H, H), par(L, H), par(L, H)
        self.ext = ext

    def forward(self, tokens, spans, max_len, seed=0, p=0.0):
        x = self.words[tokens]
        self.g, self.c = x @ self.gate, x @ self.cand
        self.h, self.last = self.ext.gated_scan(self.g, self.c, spans, max_len)
        self.k = torch.tanh(self.h @ self.key)
        self.O, self.lse = self.ext.packed_label_attention(self.k, self.h, self.query, spans, max_len, CAP, p, seed)
        return self.ext.label_logits(self.O, self.label)


def batch(layout, seed):
    from gzsl_text_amd.packed import note_spans
    spans, max_len, rows = note_spans(LENS, None if layout == 'packed' else 130, DEV)
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, VOCAB, (rows,), generator=gen).to(DEV), spans, max_len, (torch.rand(len(LENS), L, generator=gen) < 0.2).float().to(DEV)


@pytest.mark.parametrize('p', [0.0, 0.25], ids=['plain', 'dropout'])
@pytest.mark.parametrize('layout', ['packed', 'padded'])
def test_a_training_step(ops, ext, layout, p):
    """The operators' results lie within their 64-bit bounds on the inputs that the run gives them; the gradients that autograd
    hands on are, bit for bit, those of the operators' own backward entry points; the parameters move by the clipped update."""
    from gzsl_text_amd.modules.common_module import AdamW
    net = Scorer(ext, seed=1)
    opt = AdamW(list(net.parameters()), lr=1e-3, weight_decay=1e-4, max_grad_norm=0.05)
    for step in range(2):
        tokens, spans, max_len, y = batch(layout, seed=step)
        logits = net(tokens, spans, max_len, 5 + step, p)
        for t in (net.g, net.c, net.h, net.k, net.O):
            t.retain_grad()
        loss = ext.ldam_bce(logits, y)
        opt.zero_grad()
        loss.backward()
        sl = [tuple(r) for r in spans.tolist()]
        ref = scan_ref(net.g, net.c, sl)
        within(net.h, ref['h'], 'h')
        within(net.last, ref['last'], 'last')
        k, h, q = (t.detach() for t in (net.k, net.h, net.query))
        O, lse, rest = ops.attn_packed_fwd(k, h, q, spans, max_len, CAP, seed=5 + step, p=p)
        assert torch.equal(O, net.O) and torch.equal(lse, net.lse)
        if not p:
            within(O, attn_ref(k, h, q, sl, CAP)['O'], 'O')
        dk, dv, dq = ops.attn_packed_bwd(net.O.grad, O, lse, rest, k, h, q, spans, max_len, CAP, seed=5 + step, p=p)
        assert torch.equal(dk, net.k.grad) and torch.equal(dq, net.query.grad)
        # h is the keys' input and the values: its gradient is the sum of both, added by autograd
        through = (dk * (1 - k * k)) @ net.key.detach().T
        bound = (H + 8) * U * ((dk.abs() * (1 - k * k)) @ net.key.detach().abs().T) + 2 * U * (through.abs() + dv.abs())
        assert ((net.h.grad - (dv + through)).abs() <= 2 * bound).all()
        dg, dc, _ = ops.gated_scan_bwd(net.h.grad, None, h, net.g.detach(), net.c.detach(), spans, max_len)
        assert torch.equal(dg, net.g.grad) and torch.equal(dc, net.c.grad)
        before = [[t.clone() for t in ts] for ts in ([x.detach() for x in net.parameters()], [x.grad for x in net.parameters()])]
        state = [[opt.state[x][n].clone() if opt.state[x] else torch.zeros_like(x) for x in net.parameters()] for n in ('next_m', 'next_v')]
        opt.step()
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in before[1]))
        assert abs(float(opt.grad_norm) - norm) <= (U + 1e-12) * norm and norm > 0.05
        ops.adamw_clip_step_(before[0], before[1], *state, 0.05, 1e-3, 0.9, 0.999, 1e-6, 1e-4)
        for x, want in zip(net.parameters(), before[0]):
            assert torch.equal(x.detach(), want)


def test_gradients_are_the_slopes_of_the_loss(ops, ext):
    """Every parameter's gradient against central differences of the whole run in 64 bits, along one direction each.  In fp32 the
    score of a (note, label) passes through sums of at most 130 + 3 * 40 terms a stage and four stages; the loss's gradient, a
    sum over 115 of them, is taken to 2000 u of the product of norms of gradient and direction, which no cancellation inside the sums
    enters at these sizes (weights of 0.3, states below 1); the differences, of fourth order, are off by (1e-4)^4 of the fifth
    derivative along directions of norm 30 to 45 (4e-10 of it) and 1e-16 / 1e-4 of the loss, both below 1e-6 of that product."""
    net = Scorer(ext, seed=2)
    tokens, spans, max_len, y = batch('packed', seed=3)
    ext.ldam_bce(net(tokens, spans, max_len), y).backward()
    names = ('words', 'gate', 'cand', 'key', 'query', 'label')
    base = {n: getattr(net, n).detach().cpu().double() for n in names}
    tk, sl, yy = tokens.cpu(), [tuple(r) for r in spans.tolist()], y.cpu().double()

    def loss(w, on=None):
        x = w['words'][tk]
        g, c = x @ w['gate'], x @ w['cand']
        z, rows = torch.sigmoid(g), []
        for s, n in sl:
            h = torch.zeros(H, dtype=torch.float64)
            for r in range(s, s + n):
                h = (1 - z[r]) * h + z[r] * c[r]
                rows.append(h)
        h = torch.stack(rows)
        k = torch.tanh(h @ w['key'])
        out = []
        for s, n in sl:
            a = CAP * torch.tanh(w['query'] @ k[s:s + n].T / CAP)
            out.append(torch.softmax(a, 1) @ h[s:s + n] if n else torch.zeros(L, H, dtype=torch.float64))
        O = torch.stack(out)
        if on is None:
            return O > 0
        logits = (O * on * w['label']).sum(2)
        return torch.nn.functional.binary_cross_entropy_with_logits(logits, yy, reduction='sum') / len(sl)

    on = loss(base)  # the scores take relu(O): its kinks held where they are, the differences see a smooth function of the same slope
    gen = torch.Generator().manual_seed(4)
    for n in names:
        grad = getattr(net, n).grad.cpu().double()
        d = torch.randn(base[n].shape, generator=gen, dtype=torch.float64)
        at = lambda e: float(loss(dict(base, **{n: base[n] + e * d}), on))  # noqa: E731
        slope = (8 * (at(1e-4) - at(-1e-4)) - (at(2e-4) - at(-2e-4))) / 12e-4
        got = float((grad * d).sum())
        assert abs(got - slope) <= (2000 * U + 1e-6) * float(grad.norm() * d.norm()), (n, got, slope)


def test_serving_by_single_tokens_ends_where_the_scan_does(ops, ext):
    """gated_scan_step_ over a padded batch, ended notes inactive: its states are the scan's last ones, both within the bound."""
    from gzsl_text_amd.packed import note_spans
    T = max(LENS)
    spans, max_len, rows = note_spans(LENS, T, DEV)
    gen = torch.Generator().manual_seed(6)
    g, c = (torch.randn(rows, H, generator=gen).to(DEV) for _ in range(2))
    h0 = torch.randn(len(LENS), H, generator=gen).to(DEV)
    ref = scan_ref(g, c, [tuple(r) for r in spans.tolist()], h0)['last']
    within(ext.gated_scan(g, c, spans, max_len, h0)[1], ref, 'last')
    state, n = h0.clone(), torch.tensor(LENS, device=DEV)
    gt, ct = (x.view(len(LENS), T, H) for x in (g, c))
    for t in range(T):
        ext.gated_scan_step_(gt[:, t], ct[:, t], state, n > t)
    within(state, ref, 'state')


def test_a_record_of_more_rows_than_max_len_needs_and_a_larger_max_len(ext):
    """max_len may be any bound of the lengths: results do not change with it, whatever it is beyond the rows there are."""
    from gzsl_text_amd.packed import note_spans
    spans, max_len, rows = note_spans(LENS, None, DEV)
    gen = torch.Generator().manual_seed(7)
    k, v = (torch.randn(rows, H, generator=gen).to(DEV) for _ in range(2))
    q = torch.randn(200, H, generator=gen).to(DEV)
    a, b = (ext.packed_label_attention(k, v, q, spans, n)[0] for n in (rows, 2 ** 31 - 2 ** 24))
    assert torch.equal(a, b)
    a, b = (ext.gated_scan(k, v, spans, n)[0] for n in (rows, 2 ** 31 - 2 ** 24))
    assert torch.equal(a, b)
    within(a, scan_ref(k, v, [tuple(r) for r in spans.tolist()])['h'], 'h')


def test_second_derivatives_are_refused(ext):
    from gzsl_text_amd.packed import note_spans
    spans, max_len, rows = note_spans([4, 3], None, DEV)
    x = torch.randn(rows, 8, device=DEV, requires_grad=True)
    for out in (ext.gated_scan(x, x, spans, max_len)[0], ext.packed_label_attention(x, x, x, spans, max_len)[0]):
        with pytest.raises(RuntimeError, match='differentiable once'):
            torch.autograd.grad(out.sum(), x, create_graph=True)


def test_the_same_tensor_for_every_argument(ops, ext):
    """One tensor as keys, values and queries, and as gates and candidates: its gradient is the sum of the parts."""
    from gzsl_text_amd.packed import note_spans
    spans, max_len, rows = note_spans([9, 30], None, DEV)
    x = torch.randn(rows, 16, generator=torch.Generator().manual_seed(8)).to(DEV).requires_grad_()
    xd = x.detach()
    O, lse = ext.packed_label_attention(x, x, x, spans, max_len)
    got, = torch.autograd.grad(O.sum(), x)
    O2, lse2, rest = ops.attn_packed_fwd(xd, xd, xd, spans, max_len)
    parts = ops.attn_packed_bwd(torch.ones_like(O2), O2, lse2, rest, xd, xd, xd, spans, max_len)
    assert torch.equal(O, O2) and ((got - sum(parts)).abs() <= 4 * U * sum(t.abs() for t in parts)).all()
    h, _ = ext.gated_scan(x, x, spans, max_len)
    got, = torch.autograd.grad(h.sum(), x)
    parts = ops.gated_scan_bwd(torch.ones_like(h), None, h.detach(), xd, xd, spans, max_len)[:2]
    assert ((got - sum(parts)).abs() <= 4 * U * sum(t.abs() for t in parts)).all()


def test_scan_and_clipping_on_other_streams_at_once(ops):
    from gzsl_text_amd.packed import note_spans
    spans, max_len, rows = note_spans([300, 700], None, DEV)
    made = []
    for seed in (1, 2):
        gen = torch.Generator().manual_seed(seed)
        made.append([torch.randn(rows, 64, generator=gen).to(DEV) for _ in range(4)])
    want = [(ops.gated_scan_fwd(a, b, spans, max_len), [c.clone(), d.clone()]) for a, b, c, d in made]
    norms = [ops.clip_grad_norm_(x, 1.0) for _, x in want]
    torch.cuda.synchronize()
    got = []
    for (a, b, c, d), s in zip(made, (torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            got.append((ops.gated_scan_fwd(a, b, spans, max_len), ops.clip_grad_norm_([c, d], 1.0)))
    torch.cuda.synchronize()
    for (h, clipped), norm, (h2, norm2), (_, _, c, d) in zip(want, norms, got, made):
        assert torch.equal(h[0], h2[0]) and torch.equal(h[1], h2[1]) and torch.equal(norm, norm2)
        assert torch.equal(clipped[0], c) and torch.equal(clipped[1], d)


def test_overlapping_tensors_are_refused(ops, ext):
    x = torch.randn(100, device=DEV)
    kept = x.clone()
    m, v = torch.zeros(60, device=DEV), torch.zeros(60, device=DEV)
    for fn in (lambda: ops.clip_grad_norm_([x[:60], x[40:]], 1.0), lambda: ext.clip_grad_norm_([x, x], 1.0),
               lambda: ops.adamw_clip_step_([x[:60]], [x[40:]], [m], [v], 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0),
               lambda: ext.adamw_clip_step_([x[:60]], [x[40:]], [m], [v], 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0),
               lambda: ext.adamw_clip_step_([x[:60]], [torch.ones_like(m)], [m], [m], 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0)):
        with pytest.raises(RuntimeError, match='overlap'):
            fn()
    assert torch.equal(x, kept) and not m.any()
    ops.clip_grad_norm_([x[:40], x[40:]], 1e-3)  # neighbours are two tensors
