"""The gated recurrence over the range of its arguments: 16-bit tensors as exact as 32-bit sums make them, chunks of several tiles."""
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


def make(lens, H, dtype, seed, bias=-1.0, mean=0.0, first=1.0):
    from gzsl_text_amd.packed import note_spans
    table, max_len, rows = note_spans(lens, None, DEV)
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    g, c, h0, dh, dl = 1.5 * rnd(rows, H) + bias, rnd(rows, H) + mean, first * rnd(len(lens), H), rnd(rows, H), rnd(len(lens), H)
    return (g.to(dtype).to(DEV), c.to(dtype).to(DEV), table, max_len, h0.to(DEV), dh.to(dtype).to(DEV), dl.to(DEV),
            [tuple(x) for x in table.tolist()])


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
