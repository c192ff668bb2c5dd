"""Label attention over packed notes (gzsl_packed_attn_fwd / _bwd, torch.ops.gzsl.packed_label_attention) against a 64-bit
evaluation with elementwise bounds (tests/packed_ref.py), against the padded operator, and in the calls a program makes."""
import pytest
import torch

from tests.packed_ref import attn_ref, dropout_keep, within

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


def make(lens, E, F, L, dtype, seed, pitch=None, tail=0, garbage=None):
    """Inputs on the GPU and the span list; `tail` rows behind the last note, `garbage` in every row of no note."""
    from gzsl_text_amd.packed import note_spans
    table, max_len, rows = note_spans(lens, pitch, DEV)
    gen = torch.Generator().manual_seed(seed)
    R = rows + tail
    k = torch.tanh(torch.randn(R, E, generator=gen))
    v = torch.relu(torch.randn(R, F, generator=gen))
    q = 0.3 * torch.randn(L, E, generator=gen)
    do = torch.randn(len(lens), L, F, generator=gen)
    if garbage is not None:
        own = torch.zeros(R, dtype=torch.bool)
        for s, n in table.tolist():
            own[s:s + n] = True
        k[~own], v[~own] = garbage, garbage
    return [x.to(dtype).to(DEV) for x in (k, v, q, do)] + [table, max_len, [tuple(x) for x in table.tolist()]]


SHAPES = [  # lengths, E, F, L: one token, one label, tiles of 32 and workgroups of 128 met exactly and missed by one, odd widths
    ([1], 100, 200, 1), ([1, 0, 2], 8, 8, 3), ([32], 100, 200, 32), ([31, 64, 1], 100, 200, 33), ([5, 0, 33], 1, 1, 31),
    ([127, 129], 100, 200, 129), ([100, 257], 113, 208, 128), ([40, 3], 200, 200, 257), ([96], 208, 3, 40), ([70, 0], 37, 61, 300),
    ([33, 1], 112, 112, 64), ([64], 5, 208, 1),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,E,F,L', SHAPES)
@pytest.mark.parametrize('cap', [0.0, 5.0, 50.0])
def test_forward_and_backward_against_64_bits(ops, lens, E, F, L, dtype, cap):
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=len(lens) * 1000 + E + L)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, cap)
    assert O.dtype == dtype and lse.dtype == torch.float32
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, cap)
    ref = attn_ref(k, v, q, sl, cap, do)
    for name, x in (('O', O), ('lse', lse), ('dV', dv), ('dK', dk), ('dQ', dq)):
        within(x, ref[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,L,E,F', [([3001], 3, 100, 200), ([1500, 0, 700], 5, 200, 100), ([40, 9], 2001, 100, 200), ([20], 700, 200, 200)])
def test_long_axis_is_shared_out_and_joined(ops, lens, L, E, F, dtype):
    """Few labels over many tokens (token shares, joined), few tokens under many labels (label shares, joined)."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=7)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 8.0)
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 8.0)
    ref = attn_ref(k, v, q, sl, 8.0, do)
    for name, x in (('O', O), ('lse', lse), ('dV', dv), ('dK', dk), ('dQ', dq)):
        within(x, ref[name], name)
    again = (O, lse, *ops.attn_packed_bwd(do, *ops.attn_packed_fwd(k, v, q, spans, max_len, 8.0), k, v, q, spans, max_len, 8.0))
    for x, y in zip((O, lse, dk, dv, dq), again):
        assert torch.equal(x, y)  # fixed orders, no atomics


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('garbage', [float('nan'), float('inf'), torch.finfo(torch.float32).min])
def test_padded_batch_leaves_its_padding_out(ops, dtype, garbage):
    """A padded batch seen as rows, NaN, infinities or lowest values in the padding and behind the last note."""
    k, v, q, do, spans, max_len, sl = make([37, 0, 70, 1], 36, 52, 41, dtype, seed=3, pitch=75, tail=9, garbage=garbage)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 30.0)
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 30.0)
    ref = attn_ref(k, v, q, sl, 30.0, do)
    for name, x in (('O', O), ('lse', lse), ('dV', dv), ('dK', dk), ('dQ', dq)):
        within(x, ref[name], name)
    assert torch.isneginf(lse[1]).all() and not O[1].any()
    own = torch.zeros(k.shape[0], dtype=torch.bool)
    for s, n in sl:
        own[s:s + n] = True
    assert not dk[~own].any() and not dv[~own].any()  # (exact zeros)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_dropout_has_the_padded_operators_masks(ops, dtype):
    lens, E, F, L, L_total, l_off, seed, p = [50, 0, 97], 36, 52, 67, 120, 40, 77, 0.2
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=5)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 0.0, l_off, L_total, seed, p)
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 0.0, l_off, L_total, seed, p)
    ref = attn_ref(k, v, q, sl, 0.0, do, dropout_keep(sl, L, seed, p, l_off, L_total))
    for name, x in (('O', O), ('lse', lse), ('dV', dv), ('dK', dk), ('dQ', dq)):
        within(x, ref[name], name)


@pytest.mark.parametrize('p', [0.0, 0.2])
def test_full_notes_without_a_cap_agree_with_the_padded_operator(ops, p):
    """Notes of one length, cap 0: the operator the framework had.  Both are fp32 kernels within the bound of attn_ref of the same
    64-bit value, so they differ by at most twice that."""
    B, T, E, F, L, seed = 3, 150, 100, 200, 90, 9
    k, v, q, do, spans, max_len, sl = make([T] * B, E, F, L, torch.float32, seed=11)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 0.0, 0, L, seed, p)
    O2, lse2 = ops.attn_fwd(k.view(B, T, E), v.view(B, T, F), q, 0, L, seed, p)
    ref = attn_ref(k, v, q, sl, 0.0, do, dropout_keep(sl, L, seed, p) if p else None)
    within(O, (O2.cpu().double(), 2 * ref['O'][1]), 'O')
    within(lse, (lse2.cpu().double(), 2 * ref['lse'][1]), 'lse')
    g = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 0.0, 0, L, seed, p)
    g2 = [torch.zeros(B, T, E, device=DEV), torch.zeros(B, T, F, device=DEV), torch.zeros(L, E, device=DEV)]
    ops.attn_bwd(do, O2, k.view(B, T, E), v.view(B, T, F), q, lse2, 0, L, seed, p, *g2)
    for x, y, name in zip(g, g2, ('dK', 'dV', 'dQ')):
        within(x, (y.view(x.shape).cpu().double(), 2 * ref[name][1]), name)


@pytest.mark.parametrize('cap', [0.0, 2.0])
def test_gradients_are_the_slopes_of_the_forward(ops, cap):
    """Central differences of the 64-bit forward along a random direction: their error is the third derivative times
    eps^2 / 6 plus 1e-16 / eps of cancellation, below 1e-6 of the sums of magnitudes here; the kernel's own is the bound."""
    k, v, q, do, spans, max_len, sl = make([19, 33], 20, 24, 17, torch.float32, seed=21)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, cap)
    grads = dict(zip(('dK', 'dV', 'dQ'), ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, cap)))
    ref = attn_ref(k, v, q, sl, cap, do)
    gen = torch.Generator().manual_seed(2)
    base = [x.cpu().double() for x in (k, v, q)]

    def f(args):
        out = 0.0
        for b, (s, n) in enumerate(sl):
            x = args[2] @ args[0][s:s + n].T
            if cap > 0:
                x = cap * torch.tanh(x / cap)
            out += float((torch.softmax(x, 1) @ args[1][s:s + n] * do[b].cpu().double()).sum())
        return out

    for i, name in enumerate(('dK', 'dV', 'dQ')):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        eps = 1e-4
        hi, lo = list(base), list(base)
        hi[i], lo[i] = base[i] + eps * d, base[i] - eps * d
        slope = (f(hi) - f(lo)) / (2 * eps)
        got = float((grads[name].cpu().double() * d).sum())
        tol = float((ref[name][1] * d.abs()).sum()) + 1e-6 * float((ref[name][0].abs() * d.abs()).sum())
        assert abs(got - slope) <= tol, (name, got, slope, tol)


def test_scores_far_outside_the_cap_and_rising_maxima(ops):
    """Scores of +-1e4 against a cap of 3 (tanh saturates), and, uncapped, maxima that rise by more than 2^12 from tile to tile."""
    gen = torch.Generator().manual_seed(1)
    k = torch.randn(130, 8, generator=gen)
    v, q, do = torch.randn(130, 12, generator=gen), torch.randn(5, 8, generator=gen), torch.randn(1, 5, 12, generator=gen)
    from gzsl_text_amd.packed import note_spans
    spans, max_len, _ = note_spans([130], device=DEV)
    kc = (k * 1e4).to(DEV)
    O, lse, rest = ops.attn_packed_fwd(kc, v.to(DEV), q.to(DEV), spans, max_len, 3.0)
    ref = attn_ref(kc, v, q, [(0, 130)], 3.0)
    within(O, ref['O'], 'O at saturation')
    ramp = (k * torch.linspace(0.0, 12.0, 130)[:, None]).to(DEV)
    O, lse, rest = ops.attn_packed_fwd(ramp, v.to(DEV), q.to(DEV), spans, max_len)
    dk, dv, dq = ops.attn_packed_bwd(do.to(DEV), O, lse, rest, ramp, v.to(DEV), q.to(DEV), spans, max_len)
    ref = attn_ref(ramp, v, q, [(0, 130)], 0.0, do)
    for name, x in (('O', O), ('lse', lse), ('dV', dv), ('dK', dk), ('dQ', dq)):
        within(x, ref[name], name + ' with rising maxima')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_row_pitches_and_alignment(ops, ext, dtype):
    """Column slices of wider tensors (any pitch, any alignment), reversed rows and a transposed tensor (copied)."""
    k, v, q, do, spans, max_len, sl = make([33, 20], 31, 45, 37, dtype, seed=8)
    ref = attn_ref(k, v, q, sl, 4.0, do)
    for off in (0, 1, 3):
        kw, vw, qw = (torch.randn(x.shape[0], x.shape[1] + 11, device=DEV).to(dtype) for x in (k, v, q))
        ks, vs, qs = (w[:, off:off + x.shape[1]] for w, x in zip((kw, vw, qw), (k, v, q)))
        for s, x in zip((ks, vs, qs), (k, v, q)):
            s.copy_(x)
        O, lse, rest = ops.attn_packed_fwd(ks, vs, qs, spans, max_len, 4.0)
        got = (O, lse, *ops.attn_packed_bwd(do, O, lse, rest, ks, vs, qs, spans, max_len, 4.0))
        for name, x in zip(('O', 'lse', 'dK', 'dV', 'dQ'), got):
            within(x, ref[name], name)
    kt = k.t().contiguous().t()
    within(ext.packed_label_attention(kt, v, q, spans, max_len, 4.0)[0], ref['O'], 'O of transposed keys')


def test_torch_operator_and_autograd(ops, ext):
    k, v, q, do, spans, max_len, sl = make([30, 0, 45], 24, 40, 19, torch.float32, seed=13)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 6.0)
    want = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 6.0)
    a = [x.clone().requires_grad_(True) for x in (k, v, q)]
    O2, lse2 = ext.packed_label_attention(*a, spans, max_len, 6.0)
    assert torch.equal(O, O2) and torch.equal(lse, lse2) and not lse2.requires_grad
    O2.backward(do)
    for x, y in zip(a, want):
        assert torch.equal(x.grad, y)
    # an upstream gradient that is a broadcast view, and only one input that wants a gradient
    b = [k, v.clone().requires_grad_(True), q]
    ext.packed_label_attention(*b, spans, max_len, 6.0)[0].sum().backward()
    ref = attn_ref(k, v, q, sl, 6.0, torch.ones_like(do))
    within(b[1].grad, ref['dV'], 'dV of a sum')
    with torch.no_grad():
        assert torch.equal(ext.packed_label_attention(*a, spans, max_len, 6.0)[0], O)
    # labels one by one, as shards of the label axis are taken
    parts = [ext.packed_label_attention(k, v, q[i:i + 7], spans, max_len, 6.0)[0] for i in range(0, 19, 7)]
    within(torch.cat(parts, 1), attn_ref(k, v, q, sl, 6.0)['O'], 'O by label shards')


def test_captured_and_replayed_with_new_inputs(ops):
    """Forward and backward recorded into a graph; replays on refreshed inputs, with eager work between, give the eager bits."""
    k, v, q, do, spans, max_len, _ = make([40, 33], 100, 200, 65, torch.bfloat16, seed=31)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 30.0)
        ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 30.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 30.0)
        g = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 30.0)
    for seed in (1, 2, 3):
        k2, v2, q2, do2 = make([40, 33], 100, 200, 65, torch.bfloat16, seed=seed)[:4]
        for x, y in zip((k, v, q, do), (k2, v2, q2, do2)):
            x.copy_(y)
        graph.replay()
        O2, lse2, rest2 = ops.attn_packed_fwd(k2, v2, q2, spans, max_len, 30.0)
        g2 = ops.attn_packed_bwd(do2, O2, lse2, rest2, k2, v2, q2, spans, max_len, 30.0)
        torch.cuda.synchronize()
        for x, y in zip((O, lse, *g), (O2, lse2, *g2)):
            assert torch.equal(x, y)


def test_on_another_stream_and_two_at_once(ops):
    a = make([60, 61], 100, 200, 70, torch.float32, seed=41)
    b = make([60, 61], 100, 200, 70, torch.float32, seed=42)
    want = [ops.attn_packed_fwd(*x[:3], x[4], x[5], 9.0) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(ops.attn_packed_fwd(*x[:3], x[4], x[5], 9.0))
    torch.cuda.synchronize()
    for (O, lse, _), (O2, lse2, _) in zip(want, got):
        assert torch.equal(O, O2) and torch.equal(lse, lse2)


def test_empty_extents(ops, ext):
    k, v, q, do, spans, max_len, _ = make([0, 0], 8, 8, 4, torch.float32, seed=1)
    O, lse = ext.packed_label_attention(k, v, q, spans, max_len)
    assert O.shape == (2, 4, 8) and not O.any() and torch.isneginf(lse).all()
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, None, k, v, q, spans, max_len)
    assert dk.shape == (0, 8) and dv.shape == (0, 8) and not dq.any()
    none = torch.zeros((0, 2), dtype=torch.int64, device=DEV)
    x = torch.ones(3, 8, device=DEV, requires_grad=True)
    O, lse = ext.packed_label_attention(x, torch.ones(3, 8, device=DEV), q, none, 0)
    assert O.shape == (0, 4, 8)
    O.sum().backward()
    assert not x.grad.any()
    O, lse = ext.packed_label_attention(torch.ones(3, 8, device=DEV), torch.ones(3, 8, device=DEV), q[:0], torch.tensor([[0, 3]], device=DEV), 3)
    assert O.shape == (1, 0, 8)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('cap', [0.0, 30.0, 31.0])
def test_backward_from_lse_and_output_alone(ops, dtype, cap):
    """Without the forward's statistics: the rounding of lse and of O enters (their bounds, in attn_ref)."""
    k, v, q, do, spans, max_len, sl = make([70, 33], 100, 200, 90, dtype, seed=17)
    O, lse, none = ops.attn_packed_fwd(k, v, q, spans, max_len, cap, need_grad=False)
    assert none is None
    got = ops.attn_packed_bwd(do, O, lse, None, k, v, q, spans, max_len, cap)
    ref = attn_ref(k, v, q, sl, cap, do, rest=False)
    for name, x in zip(('dK', 'dV', 'dQ'), got):
        within(x, ref[name], name)


def test_many_notes(ops):
    """More notes than a wave has lanes: 200 of them, some empty, both types of cut."""
    gen = torch.Generator().manual_seed(4)
    lens = [int(x) for x in torch.randint(0, 40, (200,), generator=gen)]
    lens[77] = 700
    for L in (9, 150):
        k, v, q, do, spans, max_len, sl = make(lens, 20, 24, L, torch.float32, seed=5)
        O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 4.0)
        got = (O, lse, *ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 4.0))
        ref = attn_ref(k, v, q, sl, 4.0, do)
        for name, x in zip(('O', 'lse', 'dK', 'dV', 'dQ'), got):
            within(x, ref[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('E,cap', [(24, 0.0), (24, 30.0), (200, 0.0), (200, 3.0)])
def test_more_workgroups_than_the_chip_has_places(ops, dtype, E, cap):
    """66 notes x 1100 labels: label workgroups of full width in both directions, at both key widths."""
    gen = torch.Generator().manual_seed(6)
    lens = [int(x) for x in torch.randint(0, 50, (65,), generator=gen)] + [133]
    k, v, q, do, spans, max_len, sl = make(lens, E, 40, 1100, dtype, seed=9, tail=2)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, cap)
    got = (O, lse, *ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, cap))
    ref = attn_ref(k, v, q, sl, cap, do)
    for name, x in zip(('O', 'lse', 'dK', 'dV', 'dQ'), got):
        within(x, ref[name], name)


def test_a_wrong_table_is_clamped_to_the_rows(ops):
    """Counts and starts outside of the rows give other numbers, never an access out of range (the kernels clamp them)."""
    k, v, q, do, _, _, _ = make([40], 16, 16, 5, torch.float32, seed=2)
    bad = torch.tensor([[-5, 20], [30, 1000], [10 ** 12, 4], [3, -7]], dtype=torch.int64, device=DEV)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, bad, 64)
    ref = attn_ref(k, v, q, [(0, 20), (30, 10), (40, 0), (3, 0)])
    within(O, ref['O'], 'O')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_notes_that_overlap_stay_inside_the_workspace(ops, dtype):
    """A table of notes over the same rows: the forward and dQ, sums of whole notes, are right; dK and dV hold one note's or another's
    part (the table has to be disjoint for them), and nothing around them is touched."""
    k, v, q, do, _, _, _ = make([300], 40, 24, 70, dtype, seed=3)
    spans = torch.tensor([[0, 300]] * 40, dtype=torch.int64, device=DEV)
    do = do.expand(40, -1, -1).contiguous()
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, 300)
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, 300)
    ref = attn_ref(k, v, q, [(0, 300)] * 40, dout=do)
    within(O, ref['O'], 'O')
    within(dq, ref['dQ'], 'dQ')
    assert dk.shape == k.shape and dv.shape == v.shape


@pytest.mark.parametrize('cap', [0.0, 10.0])
@pytest.mark.parametrize('lens,E,F,L', [([40, 13, 1], 200, 200, 60), ([300, 517], 100, 200, 1), ([20], 30, 8, 300), ([700, 31], 200, 64, 150)])
def test_16_bit_gradients_are_rounded_once(ops, lens, E, F, L, cap):
    """A training call's bf16 results are the exact ones rounded, up to 32-bit sums and two-piece weights (2^-16): nothing in between is
    rounded to 16 bits, whose errors the cancellation in dS would multiply."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, torch.bfloat16, seed=11)
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, cap)
    got = (O, *ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, cap))
    ref = attn_ref(k, v, q, sl, cap, do, two=True)
    for name, x in zip(('O', 'dK', 'dV', 'dQ'), got):
        within(x, ref[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,E,F,L', [([130, 7], 30, 156, 1500), ([129], 100, 200, 900), ([20, 0, 31], 200, 33, 2100)])
def test_token_tiles_of_many_runs(ops, dtype, lens, E, F, L):
    """Few tokens, many labels: a token tile's gradients come from many workgroups' parts, odd and even widths, rows between notes."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=13, pitch=140, tail=5, garbage=float('nan'))
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, 5.0)
    got = (O, lse, *ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, 5.0))
    ref = attn_ref(k, v, q, sl, 5.0, do)
    for name, x in zip(('O', 'lse', 'dK', 'dV', 'dQ'), got):
        within(x, ref[name], name)
