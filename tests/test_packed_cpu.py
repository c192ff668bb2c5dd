"""Packed-note operators and gradient clipping without a GPU: the host plan, the schemas, the struct layouts and every refusal
(bad arguments come back as GZSL_EINVAL / an exception before anything is launched)."""
import ctypes
import os
import re

import pytest
import torch

from gzsl_text_amd import hip
from gzsl_text_amd.packed import note_spans

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def ext():
    from gzsl_text_amd import torch_ext
    torch_ext.build()
    torch_ext.load()
    return torch.ops.gzsl


def test_note_spans():
    t, n, rows = note_spans([3, 0, 5], device='cpu')
    assert t.tolist() == [[0, 3], [3, 0], [3, 5]] and n == 5 and rows == 8 and t.dtype == torch.int64
    t, n, rows = note_spans([3, 0, 5], pitch=7, device='cpu')
    assert t.tolist() == [[0, 3], [7, 0], [14, 5]] and n == 5 and rows == 21
    t, n, rows = note_spans([], device='cpu')
    assert t.shape == (0, 2) and n == 0 and rows == 0
    with pytest.raises(ValueError):
        note_spans([3, -1], device='cpu')
    with pytest.raises(ValueError):
        note_spans([3, 9], pitch=8, device='cpu')


@pytest.mark.parametrize('name', ['GzslPackedAttn', 'GzslGatedScan'])
def test_struct_layouts_match_the_header(name):
    src = open(os.path.join(ROOT, 'include', 'gzsl_hip.h')).read()
    body = re.sub(r'/\*.*?\*/', '', src[src.index('typedef struct %s {' % name):src.index('} %s;' % name)], flags=re.S)
    kinds = {'void*': ctypes.c_void_p, 'int64_t*': ctypes.c_void_p, 'float*': ctypes.c_void_p, 'long long': ctypes.c_longlong,
             'int': ctypes.c_int, 'float': ctypes.c_float, 'uint32_t': ctypes.c_uint32}
    want = []
    for decl in body.split('{', 1)[1].split(';'):
        decl = decl.replace('const ', '').strip()
        if decl:
            kind, names = re.match(r'(long long|[a-z0-9_]+\*?)\s+(.*)', decl, flags=re.S).groups()
            want += [(n.strip(), kinds[kind]) for n in names.split(',')]
    assert [tuple(f) for f in getattr(hip, name)._fields_] == want


def test_schemas(ext):
    assert str(ext.packed_label_attention.default._schema) == (
        'gzsl::packed_label_attention(Tensor keys, Tensor values, Tensor queries, Tensor spans, int max_len, float cap=0., '
        'float p_drop=0., int seed=0, int l_offset=0, int L_total=0) -> (Tensor, Tensor)')
    assert str(ext.gated_scan.default._schema) == (
        'gzsl::gated_scan(Tensor gates, Tensor cands, Tensor spans, int max_len, Tensor? h0=None, bool reverse=False) -> '
        '(Tensor, Tensor)')
    assert str(ext.clip_grad_norm_.default._schema) == 'gzsl::clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor'


def test_no_cpu_path(ext):
    t, n, rows = note_spans([3, 4], device='cpu')
    x = torch.zeros(rows, 8)
    for fn in (lambda: ext.packed_label_attention(x, x, x, t, n), lambda: ext.gated_scan(x, x, t, n),
               lambda: ext.gated_scan_step_(x, x, x), lambda: ext.clip_grad_norm_([x], 1.0),
               lambda: ext.adamw_clip_step_([x], [x], [x], [x], 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            fn()
    from gzsl_text_amd.ops_hip import HipOps
    ops = HipOps()
    for fn in (lambda: ops.attn_packed_fwd(x, x, x, t, n), lambda: ops.gated_scan_fwd(x, x, t, n),
               lambda: ops.gated_scan_step_(x, x, x.clone()), lambda: ops.clip_grad_norm_([x], 1.0)):
        with pytest.raises(RuntimeError):
            fn()


lib_built = pytest.mark.skipif(not os.path.exists(hip.LIB_PATH), reason='library not built (run __graft_entry__.build())')


def attn(**kw):
    d = dict(rows=10, ldk=8, ldv=8, ldq=8, B=2, max_len=5, L=4, E=8, F=8, dtype=hip.F32, cap=0.0, l_offset=0, L_total=4,
             drop_scale=1.0)
    d.update(kw)
    return hip.GzslPackedAttn(**d)


@lib_built
@pytest.mark.parametrize('bad', [dict(E=0), dict(E=209), dict(F=0), dict(F=209), dict(B=-1), dict(rows=-1), dict(max_len=-1), dict(L=-1),
                                 dict(dtype=2), dict(cap=-1.0), dict(cap=float('nan')), dict(cap=float('inf')), dict(ldk=7), dict(ldv=7),
                                 dict(ldq=7)])
def test_attention_refuses(bad):
    lib = hip.load()
    d = attn(**bad)
    for backward in (0, 1):
        assert lib.gzsl_packed_attn_work_bytes(d, backward) == -1
    p = ctypes.c_void_p(4096)  # never dereferenced: the arguments are refused first
    assert lib.gzsl_packed_attn_fwd(d, p, p, p, p, 1 << 40, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_bwd(d, p, p, p, p, p, p, p, p, 1 << 40, None) == hip.EINVAL


@lib_built
def test_attention_refuses_missing_pointers_and_short_workspaces():
    lib = hip.load()
    p = ctypes.c_void_p(4096)
    d = attn()
    need = lib.gzsl_packed_attn_work_bytes(d, 0)
    assert need > 0
    assert lib.gzsl_packed_attn_fwd(d, p, p, p, p, need, None) == hip.EINVAL  # no tensors
    d = attn(keys=4096, values=4096, queries=4096, spans=4096)
    assert lib.gzsl_packed_attn_fwd(d, p, p, p, p, need - 1, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_fwd(d, p, p, None, ctypes.c_void_p(4097), need, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_fwd(d, None, p, None, p, need, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_fwd(d, p, p, ctypes.c_void_p(4100), p, need, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_bwd(d, p, p, p, None, p, p, p, p, 1 << 40, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_fwd(None, p, p, p, p, need, None) == hip.EINVAL
    assert lib.gzsl_packed_attn_work_bytes(attn(B=70000), 0) == -1


@lib_built
@pytest.mark.parametrize('bad', [dict(H=0), dict(B=-1), dict(rows=-1), dict(max_len=-1), dict(ldg=7), dict(ldc=7), dict(dtype=5),
                                 dict(spans=None), dict(gates=None), dict(cands=None)])
def test_scan_refuses(bad):
    lib = hip.load()
    d = dict(gates=4096, cands=4096, spans=4096, h0=None, rows=10, ldg=8, ldc=8, B=2, max_len=5, H=8, reverse=0, dtype=hip.F32)
    d.update(bad)
    d = hip.GzslGatedScan(**d)
    p = ctypes.c_void_p(4096)
    assert lib.gzsl_gated_scan_fwd(d, p, p, p, 1 << 40, None) == hip.EINVAL
    assert lib.gzsl_gated_scan_bwd(d, p, p, p, p, p, p, p, 1 << 40, None) == hip.EINVAL
    assert lib.gzsl_gated_scan_step(p, p, p, None, 2, 8, 7, 8, hip.F32, None) == hip.EINVAL
    assert lib.gzsl_gated_scan_step(p, p, None, None, 2, 8, 8, 8, hip.F32, None) == hip.EINVAL


@lib_built
def test_clip_refuses():
    lib = hip.load()
    sizes = (ctypes.c_longlong * 2)(5, 6)
    types = (ctypes.c_int * 2)(hip.F32, hip.BF16)
    ptrs = (ctypes.c_void_p * 2)(4096, 8192)
    null = (ctypes.c_void_p * 2)(4096, None)
    p = ctypes.c_void_p(4096)
    need = lib.gzsl_clip_work_bytes(sizes, 2)
    assert need > 0
    for args in ((ptrs, sizes, types, 2, 0.0, p, p, need), (ptrs, sizes, types, 2, -1.0, p, p, need),
                 (ptrs, sizes, types, 2, float('nan'), p, p, need), (ptrs, sizes, types, 2, 1.0, None, p, need),
                 (ptrs, sizes, types, 2, 1.0, p, p, need - 1), (ptrs, sizes, types, 2, 1.0, p, None, need),
                 (null, sizes, types, 2, 1.0, p, p, need), (ptrs, sizes, types, -1, 1.0, p, p, need),
                 (ptrs, (ctypes.c_longlong * 2)(5, -6), types, 2, 1.0, p, p, need),
                 (ptrs, sizes, (ctypes.c_int * 2)(0, 3), 2, 1.0, p, p, need)):
        assert lib.gzsl_clip_grad_norm(*args, None) == hip.EINVAL
    assert lib.gzsl_clip_work_bytes((ctypes.c_longlong * 1)(-1), 1) == -1
    assert lib.gzsl_adamw_clip_step(ptrs, ptrs, ptrs, null, sizes, 2, 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0, p, p, need, None) == hip.EINVAL
    assert lib.gzsl_adamw_clip_step(ptrs, ptrs, ptrs, ptrs, sizes, 2, 0.0, 1e-3, 0.9, 0.999, 1e-6, 0.0, p, p, need, None) == hip.EINVAL


def test_adamw_refuses_a_bad_max_grad_norm():
    from gzsl_text_amd.modules.common_module import AdamW
    for bad in (0.0, -1.0, float('nan')):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], max_grad_norm=bad)


@lib_built
@pytest.mark.parametrize('cap', [1e-31, 2e30])
def test_attention_refuses_a_cap_without_a_reciprocal(cap):
    assert hip.load().gzsl_packed_attn_work_bytes(attn(cap=cap), 0) == -1


@lib_built
def test_max_len_beyond_the_rows_takes_no_more_workspace():
    lib = hip.load()
    for backward in (0, 1):
        assert lib.gzsl_packed_attn_work_bytes(attn(max_len=2 ** 30), backward) == lib.gzsl_packed_attn_work_bytes(attn(max_len=10), backward) > 0
    d = dict(gates=4096, cands=4096, spans=4096, h0=None, rows=10 ** 5, ldg=8, ldc=8, B=1, max_len=10 ** 5, H=8, reverse=0, dtype=hip.F32)
    need = lib.gzsl_gated_scan_work_bytes(hip.GzslGatedScan(**d), 0)
    assert need > 0 and lib.gzsl_gated_scan_work_bytes(hip.GzslGatedScan(**dict(d, max_len=2 ** 30)), 0) == need
    # chunk sizes stay below 2^31 at the largest batch, and a width of more channels than the grid has room for is refused
    assert lib.gzsl_gated_scan_work_bytes(hip.GzslGatedScan(**dict(d, B=65534, rows=2 ** 31, max_len=2 ** 30)), 0) >= 0
    assert lib.gzsl_gated_scan_work_bytes(hip.GzslGatedScan(**dict(d, H=65537, ldg=65537, ldc=65537)), 0) == -1


def test_overlapping_tensors_are_found():
    from gzsl_text_amd.ops_hip import HipOps
    x = torch.zeros(10)
    HipOps._apart([x[:5], x[5:], x[:0]], [torch.ones(3)])
    HipOps._apart([torch.ones(2)], [x, x])  # read twice: nothing is written there
    for written, read in (([x, x], ()), ([x[:6], x[5:]], ()), ([x[2:4]], [x]), ([x], [x[9:]]), ([x[:1], x], [x])):
        with pytest.raises(RuntimeError, match='overlap'):
            HipOps._apart(written, read)


@lib_built
@pytest.mark.parametrize('E', [100, 200])
@pytest.mark.parametrize('dtype', [hip.F32, hip.BF16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('B,rows,max_len,L', [(64, 103000, 40000, 300), (16, 55000, 40000, 300), (1000, 200000, 60000, 500)])
def test_one_long_note_among_many_takes_workspace_for_the_rows_there_are(B, rows, max_len, L, dtype, E):
    """Scratch for what is read and written: at most ten times the inputs, the output and its gradient, and the fixed shares of the
    chip's workgroups (256 pieces of a [L, F] output; 512 of 128 tokens); sized for a padded batch it was up to 60 times."""
    lib, F, w = hip.load(), 200, 4 if dtype == hip.F32 else 2
    d = attn(rows=rows, ldk=E, ldv=F, ldq=E, B=B, max_len=max_len, L=L, E=E, F=F, dtype=dtype, L_total=L)
    data = w * (rows * (E + F) + L * E + B * L * F)
    for backward in (0, 1):
        assert 0 < lib.gzsl_packed_attn_work_bytes(d, backward) < 10 * data + 4 * (256 + B) * L * max(E, F) + 8 * 256 * 128 * (E + F)


@lib_built
def test_few_labels_need_no_images():
    lib = hip.load()
    d = attn(rows=40000, B=1, max_len=40000, L=50, E=100, F=200, ldk=100, ldv=200, ldq=100, L_total=50)
    assert lib.gzsl_packed_attn_work_bytes(d, 0) < 4 * 300 * 50 * 202 + 1024


@pytest.mark.parametrize('which', [0, 1, 2], ids=['gates', 'cands', 'state'])
def test_a_step_that_autograd_would_miss_is_refused(ext, which):
    """A leaf or a result that wants a gradient, in either binding; no_grad and detached tensors pass this check (and are then
    refused for standing on the CPU)."""
    from gzsl_text_amd.ops_hip import HipOps
    for step in (ext.gated_scan_step_, HipOps().gated_scan_step_):
        for result in (False, True):
            t = [torch.zeros(2, 3) for _ in range(3)]
            t[which].requires_grad_()
            if result:
                t[which] = t[which] * 2
            with pytest.raises(RuntimeError, match='not differentiable'):
                step(*t)
            with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match='GPU|CPU|cuda|device'):
                step(*t)
            with pytest.raises((RuntimeError, NotImplementedError), match='GPU|CPU|cuda|device'):
                step(*[x.detach() for x in t])


@pytest.mark.parametrize('l_offset,L_total', [(-1, 0), (1, 0), (3, 6), (2 ** 63 - 1, 0), (0, 2 ** 31), (2 ** 32, 2 ** 32 + 4)])
def test_labels_outside_of_their_range_are_refused(l_offset, L_total):
    from gzsl_text_amd.ops_hip import HipOps
    t, n, rows = note_spans([3, 4], device='cpu')
    x = torch.zeros(rows, 8)
    with pytest.raises(RuntimeError, match='outside of'):
        HipOps().attn_packed_fwd(x, x, x[:4], t, n, l_offset=l_offset, L_total=L_total)
