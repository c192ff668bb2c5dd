"""The gated linear recurrence over packed notes (gzsl_gated_scan_fwd / _bwd / _step, torch.ops.gzsl.gated_scan) against a
64-bit loop with elementwise bounds (tests/packed_ref.py)."""
import pytest
import torch

from tests.packed_ref import U, scan_ref, within

pytestmark = pytest.mark.gpu
DEV = 'cuda'


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


def make(lens, H, dtype, seed, pitch=None, tail=0, garbage=None, bias=-1.0):
    from gzsl_text_amd.packed import note_spans
    table, max_len, rows = note_spans(lens, pitch, DEV)
    gen = torch.Generator().manual_seed(seed)
    R, B = rows + tail, len(lens)
    g, c = 1.5 * torch.randn(R, H, generator=gen) + bias, torch.randn(R, H, generator=gen)
    h0, dh, dl = torch.randn(B, H, generator=gen), torch.randn(R, H, generator=gen), torch.randn(B, H, generator=gen)
    if garbage is not None:
        own = torch.zeros(R, dtype=torch.bool)
        for s, n in table.tolist():
            own[s:s + n] = True
        for x in (g, c, dh):
            x[~own] = garbage
    return [g.to(dtype).to(DEV), c.to(dtype).to(DEV), table, max_len, h0.to(DEV), dh.to(dtype).to(DEV), dl.to(DEV),
            [tuple(x) for x in table.tolist()]]


NAMES = ('h', 'last', 'dg', 'dc', 'dh0')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('reverse', [False, True], ids=['ahead', 'back'])
@pytest.mark.parametrize('lens,H', [([1], 1), ([1, 0, 2], 3), ([31, 64, 1], 200), ([5, 0, 33], 7), ([127, 129, 65], 100), ([300], 256),
                                    ([64, 63], 5), ([1030, 17], 33), ([2049], 64), ([128, 256], 130), ([4100], 12)])
def test_forward_and_backward_against_64_bits(ops, lens, H, dtype, reverse):
    g, c, spans, max_len, h0, dh, dl, sl = make(lens, H, dtype, seed=len(lens) + H)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0, reverse)
    assert h.dtype == dtype and last.dtype == torch.float32
    got = (h, last, *ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0, reverse))
    ref = scan_ref(g, c, sl, h0, reverse, dh, dl)
    for name, x in zip(NAMES, got):
        within(x, ref[name], name)
    again = ops.gated_scan_fwd(g, c, spans, max_len, h0, reverse)
    assert torch.equal(h, again[0]) and torch.equal(last, again[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,H,reverse', [([9000, 0, 2700, 1], 200, False), ([9001], 256, True), ([27001, 400], 5, False)])
def test_notes_of_many_chunks(ops, lens, H, dtype, reverse):
    g, c, spans, max_len, h0, dh, dl, sl = make(lens, H, dtype, seed=H, tail=3)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0, reverse)
    got = (h, last, *ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0, reverse))
    ref = scan_ref(g, c, sl, h0, reverse, dh, dl)
    for name, x in zip(NAMES, got):
        within(x, ref[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('garbage', [float('nan'), float('inf')])
def test_padded_batch_leaves_its_padding_out(ops, dtype, garbage):
    g, c, spans, max_len, h0, dh, dl, sl = make([37, 0, 70, 1], 20, dtype, seed=3, pitch=75, tail=9, garbage=garbage)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
    got = (h, last, *ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0))
    ref = scan_ref(g, c, sl, h0, False, dh, dl)
    for name, x in zip(NAMES, got):
        within(x, ref[name], name)


def test_without_initial_state_and_with_half_of_the_gradients(ops):
    g, c, spans, max_len, _, dh, dl, sl = make([40, 9], 24, torch.float32, seed=5)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len)
    for a, b in ((dh, None), (None, dl)):
        got = (h, last, *ops.gated_scan_bwd(a, b, h, g, c, spans, max_len))
        ref = scan_ref(g, c, sl, None, False, a, b)
        for name, x in zip(NAMES, got):
            within(x, ref[name], name)


def test_extreme_gates(ops):
    """Gates that open or close fully (sigmoid 0 or 1 to the last bit, +-infinity among them) and closed for a whole note."""
    for value in (200.0, -200.0, float('inf'), float('-inf')):
        g, c, spans, max_len, h0, dh, dl, sl = make([70, 3], 8, torch.float32, seed=6)
        g[::2] = value
        h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
        got = (h, last, *ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0))
        ref = scan_ref(g, c, sl, h0, False, dh, dl)
        for name, x in zip(NAMES, got):
            within(x, ref[name], f'{name} at {value}')
    g, c, spans, max_len, h0, dh, dl, sl = make([3000], 8, torch.float32, seed=6, bias=-12.0)  # remembers through 3000 steps
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
    ref = scan_ref(g, c, sl, h0)
    within(h, ref['h'], 'h with long memory')


def test_a_nan_stays_in_its_channel_and_behind_its_token(ops):
    g, c, spans, max_len, h0, _, _, sl = make([200, 50], 9, torch.float32, seed=7)
    clean = ops.gated_scan_fwd(g, c, spans, max_len, h0)[0]
    c[100, 4] = float('nan')
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
    hit = torch.zeros_like(h, dtype=torch.bool)
    hit[100:200, 4] = True
    assert torch.isnan(h[hit]).all() and torch.equal(h[~hit], clean[~hit])


def test_gradients_are_the_slopes_of_the_forward(ops):
    """Central differences of the 64-bit recurrence; their own error is below 1e-6 of the sums of magnitudes (eps 1e-4)."""
    g, c, spans, max_len, h0, dh, dl, sl = make([23, 11], 6, torch.float32, seed=9)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
    grads = ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0)
    ref = scan_ref(g, c, sl, h0, False, dh, dl)
    base = [x.cpu().double() for x in (g, c, h0)]
    up, ul = dh.cpu().double(), dl.cpu().double()

    def f(a):
        r = scan_ref(a[0], a[1], sl, a[2])
        return float((r['h'][0] * up).sum() + (r['last'][0] * ul).sum())

    gen = torch.Generator().manual_seed(2)
    for i, name in enumerate(('dg', 'dc', 'dh0')):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + 1e-4 * d, base[i] - 1e-4 * d
        slope = (f(hi) - f(lo)) / 2e-4
        got = float((grads[i].cpu().double() * d).sum())
        tol = float((ref[name][1] * d.abs()).sum()) + 1e-6 * float((ref[name][0].abs() * d.abs()).sum())
        assert abs(got - slope) <= tol, (name, got, slope, tol)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_row_pitches_and_alignment(ops, dtype):
    g, c, spans, max_len, h0, dh, dl, sl = make([33, 20], 40, dtype, seed=8)
    ref = scan_ref(g, c, sl, h0, True, dh, dl)
    for off in (0, 1, 8):
        gw, cw = (torch.randn(g.shape[0], 55, device=DEV).to(dtype) for _ in range(2))
        gs, cs = gw[:, off:off + 40], cw[:, off:off + 40]
        gs.copy_(g)
        cs.copy_(c)
        h, last = ops.gated_scan_fwd(gs, cs, spans, max_len, h0, True)
        got = (h, last, *ops.gated_scan_bwd(dh, dl, h, gs, cs, spans, max_len, h0, True))
        for name, x in zip(NAMES, got):
            within(x, ref[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('B,H', [(1, 1), (64, 200), (33, 7), (300, 256)])
def test_step_form(ops, ext, dtype, B, H):
    """One token at a time equals the recurrence's formula; ended notes keep their state, bit for bit."""
    gen = torch.Generator().manual_seed(B + H)
    g, c = (torch.randn(B, H, generator=gen).to(dtype).to(DEV) for _ in range(2))
    state = torch.randn(B, H, generator=gen).to(DEV)
    active = (torch.rand(B, generator=gen) < 0.7).to(DEV)
    old = state.clone()
    version = state._version
    ext.gated_scan_step_(g, c, state, active)
    assert state._version > version
    gd, cd, s = g.cpu().double(), c.cpu().double(), old.cpu().double()
    t1, t2 = torch.sigmoid(-gd) * s, torch.sigmoid(gd) * cd
    on = active.cpu()
    # the gates: a few roundings and the rounded exponent's |g| u; bf16 tensors take 1 - z, off by u of 1
    tol = (8 + gd.abs()) * U * (t1.abs() + t2.abs()) + U * (t1 + t2).abs() + (2 * U * s.abs() if dtype == torch.bfloat16 else 0)
    within(state[active], ((t1 + t2)[on], tol[on]), 'state')
    assert torch.equal(state[~active], old[~active])
    s2 = old.clone()
    ops.gated_scan_step_(g, c, s2, active)
    assert torch.equal(s2, state)
    s3, s4 = old.clone(), old.clone()
    ext.gated_scan_step_(g, c, s3)
    ops.gated_scan_step_(g, c, s4, torch.ones(B, dtype=torch.bool, device=DEV))
    assert torch.equal(s3, s4)


def test_steps_follow_the_scan(ops):
    """Serving token by token ends in the state the scan ends in: both are within their bound of the same 64-bit value."""
    T, B, H = 30, 4, 48
    g, c, spans, max_len, h0, _, _, sl = make([T] * B, H, torch.float32, seed=12)
    _, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
    state = h0.clone()
    for t in range(T):
        ops.gated_scan_step_(g.view(B, T, H)[:, t], c.view(B, T, H)[:, t], state)  # (strided rows)
    ref = scan_ref(g, c, sl, h0)
    within(last, ref['last'], 'scan')
    within(state, ref['last'], 'steps')


def test_torch_operator_and_autograd(ops, ext):
    g, c, spans, max_len, h0, dh, dl, sl = make([30, 0, 45], 24, torch.float32, seed=13)
    h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0, True)
    want = ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0, True)
    a = [x.clone().requires_grad_(True) for x in (g, c, h0)]
    h2, last2 = ext.gated_scan(a[0], a[1], spans, max_len, a[2], True)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    torch.autograd.backward((h2, last2), (dh, dl))
    for x, y in zip(a, want):
        assert torch.equal(x.grad, y)
    b = [x.clone().requires_grad_(True) for x in (g, c)]  # only the states are used, no initial state
    ext.gated_scan(b[0], b[1], spans, max_len)[0].sum().backward()
    ref = scan_ref(g, c, sl, None, False, torch.ones_like(dh))
    within(b[0].grad, ref['dg'], 'dg of a sum')
    within(b[1].grad, ref['dc'], 'dc of a sum')


def test_captured_and_replayed_with_new_inputs(ops):
    lens, H = [700, 33], 100
    g, c, spans, max_len, h0, dh, dl, _ = make(lens, H, torch.float32, seed=31)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
        ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, last = ops.gated_scan_fwd(g, c, spans, max_len, h0)
        grads = ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0)
    for seed in (1, 2, 3):
        new = make(lens, H, torch.float32, seed=seed)
        for x, y in zip((g, c, h0, dh, dl), (new[0], new[1], new[4], new[5], new[6])):
            x.copy_(y)
        graph.replay()
        h2, last2 = ops.gated_scan_fwd(new[0], new[1], spans, max_len, new[4])
        g2 = ops.gated_scan_bwd(new[5], new[6], h2, new[0], new[1], spans, max_len, new[4])
        torch.cuda.synchronize()
        for x, y in zip((h, last, *grads), (h2, last2, *g2)):
            assert torch.equal(x, y)


def test_empty_extents(ops, ext):
    z = torch.zeros(0, 8, device=DEV)
    spans = torch.zeros((2, 2), dtype=torch.int64, device=DEV)
    h0 = torch.randn(2, 8, device=DEV)
    h, last = ext.gated_scan(z, z, spans, 0, h0)
    assert h.shape == (0, 8) and torch.equal(last, h0)
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    h, last = ext.gated_scan(x, x.detach(), torch.zeros((0, 2), dtype=torch.int64, device=DEV), 0)
    assert not h.any() and last.shape == (0, 8)
    h.sum().backward()
    assert not x.grad.any()
    bad = torch.tensor([[-5, 2], [2, 1000], [10 ** 12, 4]], dtype=torch.int64, device=DEV)
    h, last = ops.gated_scan_fwd(x.detach(), x.detach(), bad, 64)
    ref = scan_ref(x.detach(), x.detach(), [(0, 2), (2, 1), (3, 0)])
    within(h, ref['h'], 'h of a clamped table')
