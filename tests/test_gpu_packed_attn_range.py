"""Packed label attention over the range of its arguments."""
import pytest
import torch

from tests.packed_ref import attn_ref, dropout_keep, within
from tests.packed_ref_range import attn_ref_range

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BOTH = pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])


@pytest.fixture(scope='module')
def ops():
    from gzsl_text_amd.ops_hip import HipOps
    return HipOps()


def make(lens, E, F, L, dtype, seed, tail=0, scale=0.3):
    from gzsl_text_amd.packed import note_spans
    table, max_len, rows = note_spans(lens, None, DEV)
    gen = torch.Generator().manual_seed(seed)
    k, v = torch.randn(rows + tail, E, generator=gen), torch.randn(rows + tail, F, generator=gen)
    q, do = scale * torch.randn(L, E, generator=gen), torch.randn(len(lens), L, F, generator=gen)
    return [x.to(dtype).to(DEV) for x in (k, v, q, do)] + [table, max_len, [tuple(x) for x in table.tolist()]]


def run(ops, k, v, q, do, spans, max_len, cap=0.0, **drop):
    O, lse, rest = ops.attn_packed_fwd(k, v, q, spans, max_len, cap, **drop)
    dk, dv, dq = ops.attn_packed_bwd(do, O, lse, rest, k, v, q, spans, max_len, cap, **drop)
    return dict(O=O, lse=lse, dV=dv, dK=dk, dQ=dq)


@pytest.mark.parametrize('cap', [0.0, 10.0])
@pytest.mark.parametrize('lens,E,F,L', [([40, 13, 1], 200, 200, 60), ([300, 517], 100, 200, 200), ([900], 30, 64, 9), ([70, 3], 36, 52, 1500)])
def test_16_bit_scoring_is_rounded_once(ops, lens, E, F, L, cap):
    """A call that no backward follows is as exact as one of a training step: the exact values rounded, up to 32-bit sums and weights in
    two pieces (2^-16).  Values of both signs: where a row cancels, weights rounded to 8 bits show."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, torch.bfloat16, seed=4)
    O, lse, _ = ops.attn_packed_fwd(k, v, q, spans, max_len, cap, need_grad=False)
    ref = attn_ref(k, v, q, sl, cap, two=True)
    within(O, ref['O'], 'O')
    within(lse, ref['lse'], 'lse')
    assert torch.equal(O, ops.attn_packed_fwd(k, v, q, spans, max_len, cap)[0])


@BOTH
@pytest.mark.parametrize('lens,E,F,L', [([150, 31, 1], 100, 200, 40), ([77, 0, 130], 200, 64, 150)])
@pytest.mark.parametrize('cap', [1e2, 1e3, 1e5, 1e6, 1e8, 1e30])
def test_caps_far_above_the_scores(ops, lens, E, F, L, dtype, cap):
    """Scores of deviation 3 and more under caps up to the largest that is accepted: an error relative to the score, whatever the cap."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=6)
    got, ref = run(ops, k, v, q, do, spans, max_len, cap), attn_ref_range(k, v, q, sl, cap, do)
    for name, x in got.items():
        within(x, ref[name], f'{name} at cap {cap:g}')


@BOTH
@pytest.mark.parametrize('cap', [1e-30, 1e-3, 64.0, 65.0, 300.0])
def test_caps_below_and_about_the_scores(ops, dtype, cap):
    """Scores up to twenty times the cap and far beyond it."""
    k, v, q, do, spans, max_len, sl = make([130, 40], 36, 52, 41, dtype, seed=8, scale=20.0)
    got, ref = run(ops, k, v, q, do, spans, max_len, cap), attn_ref_range(k, v, q, sl, cap, do)
    for name in ('O', 'lse', 'dV'):
        within(got[name], ref[name], f'{name} at cap {cap:g}')


@BOTH
@pytest.mark.parametrize('E,L', [(36, 150), (113, 150), (200, 1100)])
def test_one_long_note_among_many(ops, dtype, E, L):
    """Notes of very different lengths: token images are numbered by rows, not by the longest note."""
    gen = torch.Generator().manual_seed(3)
    lens = [int(x) for x in torch.randint(0, 40, (70,), generator=gen)]
    lens[41], lens[42] = 901, 64
    k, v, q, do, spans, max_len, sl = make(lens, E, 52, L, dtype, seed=12, tail=3)
    got, ref = run(ops, k, v, q, do, spans, max_len, 6.0), attn_ref_range(k, v, q, sl, 6.0, do)
    for name, x in got.items():
        within(x, ref[name], name)


@BOTH
@pytest.mark.parametrize('lens,E,F,L', [([150, 31, 1], 100, 64, 33), ([40, 70], 112, 52, 150), ([150, 31], 113, 52, 33), ([77, 0, 130], 200, 64, 300)])
@pytest.mark.parametrize('value', ['infinite', 'lowest'])
def test_tokens_masked_by_a_column_of_the_keys(ops, lens, E, F, L, dtype, value):
    """A column in which every query has 1 and a masked token's key minus infinity or the type's lowest value: its weight and its gradients
    are 0, those of the others the exact ones.  A note's last token, a note's first ones, every second one."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=14)
    low = float('-inf') if value == 'infinite' else torch.finfo(dtype).min
    q[:, -1], k[:, -1] = 1, 0
    for s, n in sl:
        k[s:s + n // 4, -1] = low
        if n > 1:
            k[s + n - 1, -1] = low
        k[s + n // 2:s + 3 * n // 4:2, -1] = low
    got, ref = run(ops, k, v, q, do, spans, max_len), attn_ref_range(k, v, q, sl, 0.0, do)
    for name in ('O', 'lse', 'dV', 'dK'):
        within(got[name], ref[name], name)
    within(got['dQ'][:, :-1], [x[:, :-1] for x in ref['dQ']], 'dQ')  # (of the column: 0 times infinity)
    out = k[:, -1] == low
    assert not got['dK'][out].any() and not got['dV'][out].any()


@BOTH
@pytest.mark.parametrize('E,L', [(36, 32), (100, 33), (112, 200), (113, 33), (200, 200)])
def test_infinite_keys_under_a_cap(ops, E, L, dtype):
    """An infinite element of a key, or of a query, is a score of +-cap: everything but the gradients that multiply it is exact."""
    k, v, q, do, spans, max_len, sl = make([70, 33], E, 40, L, dtype, seed=15)
    for x in (k, q):
        x[x == 0] = 0.5  # (0 times infinity is no number)
    k[3, 1], k[40, 5], k[69, 1], k[80, 0] = float('inf'), float('-inf'), float('inf'), float('-inf')
    ref = attn_ref_range(k, v, q, sl, 7.0, do)
    got = run(ops, k, v, q, do, spans, max_len, 7.0)
    rest = [e for e in range(E) if e not in (0, 1, 5)]
    for name in ('O', 'lse', 'dV', 'dK'):
        within(got[name], ref[name], name)
    within(got['dQ'][:, rest], [x[:, rest] for x in ref['dQ']], 'dQ')
    k, v, q, do, spans, max_len, sl = make([70, 33], E, 40, L, dtype, seed=16)
    for x in (k, q):
        x[x == 0] = 0.5
    q[0, 2], q[L - 1, 2], q[L // 2, 4] = float('inf'), float('-inf'), float('-inf')
    ref = attn_ref_range(k, v, q, sl, 7.0, do)
    got = run(ops, k, v, q, do, spans, max_len, 7.0)
    for name in ('O', 'lse', 'dV', 'dQ'):
        within(got[name], ref[name], name + ' of infinite queries')


@BOTH
@pytest.mark.parametrize('E,L', [(100, 33), (100, 200), (200, 33), (200, 200)])
def test_infinite_values(ops, E, L, dtype):
    """An infinite value makes its column of the note's rows infinite, and nothing else."""
    k, v, q, do, spans, max_len, sl = make([70, 33], E, 40, L, dtype, seed=17)
    v[5, 3], v[90, 11] = float('inf'), float('-inf')
    O, lse, _ = ops.attn_packed_fwd(k, v, q, spans, max_len, 7.0, need_grad=False)
    ref = attn_ref_range(k, v, q, sl, 7.0)
    assert torch.isposinf(O[0, :, 3]).all() and torch.isneginf(O[1, :, 11]).all()
    within(O, ref['O'], 'O')
    within(lse, ref['lse'], 'lse')


@BOTH
@pytest.mark.parametrize('lens,E,F,L', [([70, 33, 40], 100, 40, 33), ([130, 33, 60], 112, 40, 150), ([70, 33], 113, 52, 33), ([40, 400, 1], 200, 64, 300), ([33, 900], 36, 20, 5)])
@pytest.mark.parametrize('rest', [True, False], ids=['rest', 'lse'])
def test_notes_whose_tokens_are_all_masked(ops, lens, E, F, L, dtype, rest):
    """Of minus infinity nothing is left: like a note of no tokens, O = 0, lse = minus infinity and gradients of 0.  The lowest value is a
    score like any other.  The other notes do not see it."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=18)
    q[:, -1], k[:, -1] = 1, 0
    s, n = sl[1]
    other = [i for i in range(len(lens)) if i != 1]
    outside = [(0, 0) if i == 1 else x for i, x in enumerate(sl)]
    for low in (float('-inf'), torch.finfo(dtype).min):
        k[s:s + n, -1] = low
        O, lse, kept = ops.attn_packed_fwd(k, v, q, spans, max_len)
        dk, dv, dq = ops.attn_packed_bwd(do, O, lse, kept if rest else None, k, v, q, spans, max_len)
        ref = attn_ref_range(k, v, q, outside, 0.0, do)
        within(O[other], [x[other] for x in ref['O']], 'O')
        within(lse[other], [x[other] for x in ref['lse']], 'lse')
        for i in other if rest else ():
            r = slice(sl[i][0], sl[i][0] + sl[i][1])
            within(dk[r], [x[r] for x in ref['dK']], 'dK')
            within(dv[r], [x[r] for x in ref['dV']], 'dV')
        if low == float('-inf'):
            assert not O[1].any() and torch.isneginf(lse[1]).all() and not dk[s:s + n].any() and not dv[s:s + n].any()
            assert not torch.isnan(dq[:, :-1]).any()
            if rest:
                within(dq[:, :-1], [x[:, :-1] for x in ref['dQ']], 'dQ')
        else:
            # A score of 3.4e38 is off by up to (E + 2) u of it, 2e33 and more, as any sum of E products is (two of these scores, equal in
            # 64 bits, may differ by a rounding of 2e31): which tokens carry the weight is not determined, only that the weights
            # are finite, not negative and sum to 1.  O lies among the note's values, and dV sums over the tokens to the sum of dO.
            step, tol = torch.finfo(dtype).eps / 2, (2 * n + L + 20) * 2.0 ** -24 + 2.0 ** -16 * (dtype == torch.bfloat16)
            vd, g = v[s:s + n].cpu().double(), do[1].cpu().double()
            slack = (step + 2 * tol) * vd.abs().amax(0)
            x = O[1].cpu().double()
            assert (x >= vd.amin(0) - slack).all() and (x <= vd.amax(0) + slack).all()
            if rest:
                got, up = dv[s:s + n].cpu().double(), g.sum(0)
                assert ((got.sum(0) - up).abs() <= tol * g.abs().sum(0) + step * got.abs().sum(0)).all()


def any_order(lens, seed, lead=5):
    """A table of notes in no order, rows of no note in front, between and behind, notes of no tokens anywhere in it."""
    from random import Random
    r = Random(seed)
    at, spans = lead, []
    for n in lens:
        spans.append((at, n))
        at += n + r.choice([0, 0, 1, 7, 150])
    spans = [(r.choice([0, at // 2, at, s]) if n == 0 else s, n) for s, n in spans]
    r.shuffle(spans)
    return torch.tensor(spans, dtype=torch.int64, device=DEV), spans, at + 11


@BOTH
@pytest.mark.parametrize('lens,E,L', [([130, 0, 33, 257, 0, 1], 100, 40), ([130, 0, 33, 257, 0, 1], 36, 300), ([64, 32, 128], 200, 33)])
def test_a_table_in_any_order(ops, dtype, lens, E, L):
    """Notes sorted by anything: every note's results are its own, and rows of no note, which hold NaN, get zeros."""
    spans, sl, R = any_order(lens, seed=2)
    gen = torch.Generator().manual_seed(5)
    k, v = torch.full((R, E), float('nan')), torch.full((R, 52), float('nan'))
    for s, n in sl:
        k[s:s + n], v[s:s + n] = torch.randn(n, E, generator=gen), torch.randn(n, 52, generator=gen)
    k, v, q, do = (x.to(dtype).to(DEV) for x in (k, v, 0.3 * torch.randn(L, E, generator=gen), torch.randn(len(lens), L, 52, generator=gen)))
    got, ref = run(ops, k, v, q, do, spans, max(lens), 5.0), attn_ref_range(k, v, q, sl, 5.0, do)
    for name, x in got.items():
        within(x, ref[name], name)
    own = torch.zeros(R, dtype=torch.bool)
    for s, n in sl:
        own[s:s + n] = True
    assert not got['dK'][~own].any() and not got['dV'][~own].any()


@BOTH
def test_many_notes_in_any_order(ops, dtype):
    """Hundreds of notes, images by rows: one of 700 tokens among them."""
    gen = torch.Generator().manual_seed(7)
    lens = [int(x) for x in torch.randint(0, 20, (300,), generator=gen)] + [700]
    spans, sl, R = any_order(lens, seed=3)
    k, v = torch.randn(R, 36, generator=gen).to(dtype).to(DEV), torch.randn(R, 20, generator=gen).to(dtype).to(DEV)
    q, do = (0.3 * torch.randn(150, 36, generator=gen)).to(dtype).to(DEV), torch.randn(len(lens), 150, 20, generator=gen).to(dtype).to(DEV)
    got, ref = run(ops, k, v, q, do, spans, 700), attn_ref_range(k, v, q, sl, 0.0, do)
    for name, x in got.items():
        within(x, ref[name], name)


@BOTH
@pytest.mark.parametrize('lens,L', [([900], 9), ([400, 700], 150), ([70], 9)])
def test_a_value_that_is_no_number_shows_wherever_its_weight_is(ops, lens, L, dtype):
    """A weight of 0 times NaN is NaN, in a note that is cut into chunks as in one that is not: in every label's row, in that column."""
    k, v, q, do, spans, max_len, sl = make(lens, 36, 20, L, dtype, seed=21)
    q[:, -1], k[:, -1] = 1, 0
    s, n = sl[0]
    v[s + 3, 7] = float('nan')  # at a weight of e^-10000
    k[s:s + n // 2, -1] = -1e4  # (and chunks of such weights alone)
    O = ops.attn_packed_fwd(k, v, q, spans, max_len, need_grad=False)[0]
    assert torch.isnan(O[0, :, 7]).all() and torch.isnan(O).sum() == L


@BOTH
@pytest.mark.parametrize('cap', [0.0, 5.0, 100.0])
@pytest.mark.parametrize('lens,E,F,L', [([130, 0, 33], 36, 52, 150), ([900, 70], 100, 64, 300), ([900, 70], 200, 200, 150), ([33, 500], 200, 61, 40),
                                        ([40, 9], 113, 20, 1300)])
def test_dropout_in_every_form(ops, lens, E, F, L, dtype, cap):
    """Weights dropped by the counter hash, in the form of few labels and of many, at both key widths, in notes that are cut, with labels
    that are a shard of more, under no cap, the closed form and the series."""
    k, v, q, do, spans, max_len, sl = make(lens, E, F, L, dtype, seed=22)
    drop = dict(l_offset=37, L_total=L + 50, seed=4321, p=0.2)
    got = run(ops, k, v, q, do, spans, max_len, cap, **drop)
    ref = attn_ref_range(k, v, q, sl, cap, do, dropout_keep(sl, L, 4321, 0.2, 37, L + 50))
    for name, x in got.items():
        within(x, ref[name], name)


@BOTH
@pytest.mark.parametrize('E,cap', [(36, 5.0), (200, 0.0), (200, 5.0)])
def test_dropout_with_more_workgroups_than_the_chip_has_places(ops, dtype, E, cap):
    gen = torch.Generator().manual_seed(6)
    lens = [int(x) for x in torch.randint(0, 40, (65,), generator=gen)] + [133]
    k, v, q, do, spans, max_len, sl = make(lens, E, 24, 1100, dtype, seed=23)
    got = run(ops, k, v, q, do, spans, max_len, cap, seed=99, p=0.5)
    ref = attn_ref_range(k, v, q, sl, cap, do, dropout_keep(sl, 1100, 99, 0.5))
    for name, x in got.items():
        within(x, ref[name], name)


@pytest.mark.parametrize('l_offset,L_total', [(-1, 0), (1, 0), (3, 6), (2 ** 63 - 1, 0), (2 ** 63 - 4, 5), (0, 2 ** 31)])
def test_labels_outside_of_their_range_are_refused(l_offset, L_total):
    from gzsl_text_amd import torch_ext
    torch_ext.load()
    k, v, q, do, spans, max_len, sl = make([5], 8, 8, 4, torch.float32, seed=1)
    with pytest.raises(RuntimeError, match='outside of L_total'):
        torch.ops.gzsl.packed_label_attention(k, v, q, spans, max_len, 0.0, 0.0, 0, l_offset, L_total)
