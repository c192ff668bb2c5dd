"""The gated recurrence over the range of its arguments: 16-bit tensors as exact as 32-bit sums make them, chunks of several tiles."""
import pytest
import torch

from tests.packed_ref import U, half_step, scan_ref, within

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


def make(lens, H, dtype, seed, bias=-1.0, mean=0.0, first=1.0):
    from gzsl_text_amd.packed import note_spans
    table, max_len, rows = note_spans(lens, None, DEV)
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    g, c, h0, dh, dl = 1.5 * rnd(rows, H) + bias, rnd(rows, H) + mean, first * rnd(len(lens), H), rnd(rows, H), rnd(len(lens), H)
    return (g.to(dtype).to(DEV), c.to(dtype).to(DEV), table, max_len, h0.to(DEV), dh.to(dtype).to(DEV), dl.to(DEV),
            [tuple(x) for x in table.tolist()])


def ref_once(g, c, sl, h0, reverse, dh, dl):
    """scan_ref for results that are rounded to the tensors' type once, at the end: the bounds of the same numbers as fp32 tensors, that
    rounding, and in dgates the state in front of a step as it is kept for the backward, in two pieces (off by half_step^2)."""
    step = half_step(g.dtype)
    ref = scan_ref(g.float(), c.float(), sl, h0, reverse, dh.float(), dl)
    if g.dtype == torch.float32:
        return ref
    h, dc = ref['h'][0], ref['dc'][0]
    before = torch.zeros_like(h)
    for b, (s, n) in enumerate(sl):
        if n:
            rows = h[s:s + n].flip(0) if reverse else h[s:s + n]
            x = torch.cat([h0[b:b + 1].cpu().double(), rows[:-1]])
            before[s:s + n] = x.flip(0) if reverse else x
    extra = dict(dg=dc.abs() * torch.sigmoid(-g.detach().cpu().double()) * before.abs() * step * step)
    for name in ('h', 'dg', 'dc'):
        val, err = ref[name]
        err = err + extra.get(name, 0.0)
        ref[name] = (val, err + (val.abs() + err) * step)
    return ref


@pytest.mark.parametrize('reverse', [False, True], ids=['ahead', 'back'])
@pytest.mark.parametrize('lens,H,mean,bias', [([70, 0, 31], 40, 3.0, -1.0), ([300, 45], 7, 3.0, 1.0), ([700], 100, 0.0, -1.0), ([129, 64], 64, 10.0, 0.0),
                                              ([2100], 16, 3.0, -1.0)])
def test_16_bit_gradients_are_rounded_once(ops, ext, lens, H, mean, bias, reverse):
    """Candidates off centre: the state settles near them, and c - h_{t-1} in the gate's gradient cancels."""
    g, c, spans, max_len, h0, dh, dl, sl = make(lens, H, torch.bfloat16, 3, bias, mean)
    ref = ref_once(g, c, sl, h0, reverse, dh, dl)
    a = [x.clone().requires_grad_(True) for x in (g, c, h0)]
    h, last = ext.gated_scan(a[0], a[1], spans, max_len, a[2], reverse)
    torch.autograd.backward((h, last), (dh, dl))
    for name, x in zip(('h', 'last', 'dg', 'dc', 'dh0'), (h, last, *[t.grad for t in a])):
        within(x, ref[name], name)
    # the explicit pair: with what the forward kept, and without it (the backward then runs the forward for it)
    h, last, rest = ops.gated_scan_fwd(g, c, spans, max_len, h0, reverse, need_grad=True)
    for kept in (rest, None):
        for x, t in zip(ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0, reverse, kept), a):
            assert torch.equal(x, t.grad)


def test_a_far_state_through_open_gates(ops, ext):
    """1 - z to its own size, for 16-bit tensors too: a large state that open gates let decay."""
    for dtype in (torch.float32, torch.bfloat16):
        g, c, spans, max_len, h0, dh, dl, sl = make([9, 3], 24, dtype, 5, bias=10.0, first=1e4)
        h, last = ops.gated_scan_fwd(g[:12:3].contiguous(), c[:12:3].contiguous(), torch.tensor([[0, 3], [3, 1]], device=DEV), 3, h0)
        ref = scan_ref(g[:12:3].float(), c[:12:3].float(), [(0, 3), (3, 1)], h0)
        within(last, ref['last'], 'last')
        state = h0.clone()
        ext.gated_scan_step_(g[:2], c[:2], state)
        gd, cd, s = g[:2].cpu().double(), c[:2].cpu().double(), h0.cpu().double()
        t1, t2 = torch.sigmoid(-gd) * s, torch.sigmoid(gd) * cd
        within(state, (t1 + t2, (8 + gd.abs()) * U * (t1.abs() + t2.abs()) + U * (t1 + t2).abs()), 'state')


@pytest.mark.parametrize('reverse', [False, True], ids=['ahead', 'back'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,H', [([130, 0, 33, 257, 0, 1], 200), ([70, 900, 0, 31], 5), ([12, 0, 3] * 24, 40), ([3, 0, 1, 0, 7] * 60 + [300], 7)])
def test_a_table_in_any_order(ops, dtype, lens, H, reverse):
    """Notes sorted by anything, more of them than a wave has lanes and than a workgroup looks through: every note's results are its
    own, and rows of no note, which hold NaN, get zeros.  The same notes in ascending order give the same bits."""
    from tests.test_gpu_packed_attn_range import any_order
    spans, sl, R = any_order(lens, seed=4)
    gen = torch.Generator().manual_seed(5)
    g, c, dh = (torch.full((R, H), float('nan')) for _ in range(3))
    for s, n in sl:
        g[s:s + n], c[s:s + n], dh[s:s + n] = (torch.randn(n, H, generator=gen) for _ in range(3))
    g, c, dh = (x.to(dtype).to(DEV) for x in (g, c, dh))
    h0, dl = (torch.randn(len(lens), H, generator=gen).to(DEV) for _ in range(2))
    own = torch.zeros(R, dtype=torch.bool)
    for s, n in sl:
        own[s:s + n] = True
    ref = ref_once(g, c, sl, h0, reverse, torch.where(own.to(DEV)[:, None], dh, 0), dl)
    order = sorted(range(len(sl)), key=lambda i: sl[i])
    for at in (list(range(len(sl))), order):
        t, h00, dl0 = spans[at].contiguous(), h0[at].contiguous(), dl[at].contiguous()
        h, last, rest = ops.gated_scan_fwd(g, c, t, max(lens), h00, reverse, need_grad=True)
        got = (h, last, *ops.gated_scan_bwd(dh, dl0, h, g, c, t, max(lens), h00, reverse, rest))
        for name, x in zip(('h', 'last', 'dg', 'dc', 'dh0'), got):
            within(x, [y[at] for y in ref[name]] if name in ('last', 'dh0') else ref[name], name)
        for x in (got[0], got[2], got[3]):
            assert not x[~own].any()
        first = got if at is not order else first
    for i in (0, 2, 3):
        assert torch.equal(first[i], got[i])


@pytest.mark.parametrize('reverse', [False, True], ids=['ahead', 'back'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('lens,H', [([1100, 0, 33, 700, 64, 31, 1, 1057], 2048), ([1701, 700, 64, 1, 0, 33, 96, 1500], 257), ([1400, 96, 65, 31], 4100)])
def test_chunks_of_several_tiles(ops, dtype, lens, H, reverse):
    """Wide states make chunks of two tiles and more; notes end in a chunk's first tile, at its end, inside its last one."""
    g, c, spans, max_len, h0, dh, dl, sl = make(lens, H, dtype, seed=8)
    h, last, rest = ops.gated_scan_fwd(g, c, spans, max_len, h0, reverse, need_grad=True)
    got = (h, last, *ops.gated_scan_bwd(dh, dl, h, g, c, spans, max_len, h0, reverse, rest))
    ref = ref_once(g, c, sl, h0, reverse, dh, dl)
    for name, x in zip(('h', 'last', 'dg', 'dc', 'dh0'), got):
        within(x, ref[name], name)
