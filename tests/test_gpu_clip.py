"""Global gradient norm, clipping and the clipped AdamW update (gzsl_clip_grad_norm, gzsl_adamw_clip_step) against 64 bits.
u = 2^-24 is half a step of fp32; the squares are added in 64 bits, so the norm is off by its own last rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


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


def tensors(sizes, kinds, seed, scale=0.02):
    gen = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=gen)).to(k).to(DEV) for n, k in zip(sizes, kinds)]


def factor(norm, max_norm):
    max_norm = float(torch.tensor(max_norm, dtype=torch.float32))  # the entry points take it as a C float
    return min(1.0, max_norm / (norm + 1e-6))


def norm64(grads):
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


F32, BF16 = torch.float32, torch.bfloat16
LISTS = [  # one element, empty tensors among others, odd sizes, shares met exactly and missed by one, more than a launch holds
    ([1], [F32]), ([0, 7, 0], [F32, BF16, BF16]), ([16384, 16385, 16383], [F32] * 3), ([3, 100001, 50, 8], [BF16, F32, BF16, F32]),
    ([i % 17 + 1 for i in range(150)], [F32, BF16] * 75), ([300000] * 3, [BF16] * 3),
]


@pytest.mark.parametrize('sizes,kinds', LISTS)
@pytest.mark.parametrize('max_norm', [1e-3, 0.7, 1e9, float('inf')])
def test_clip_against_64_bits(ops, ext, sizes, kinds, max_norm):
    base = tensors(sizes, kinds, seed=len(sizes))
    n = norm64(base)
    f = factor(n, max_norm)
    results = []
    for fn in (ops.clip_grad_norm_, ext.clip_grad_norm_):
        g = [x.clone() for x in base]
        norm = fn(g, max_norm)
        assert norm.shape == () and norm.dtype == F32
        assert abs(float(norm) - n) <= (U + 1e-12) * n
        for x, y in zip(base, g):
            want = x.double() * f
            # f and the product are rounded to fp32, bf16 gradients once more to their type
            tol = want.abs() * (2.1 * U + (2.0 ** -8 if x.dtype == BF16 else 0.0)) + (2.0 ** -134 if x.dtype == BF16 else 2.0 ** -149)
            assert ((y.double() - want).abs() <= tol).all()
            if f == 1.0:
                assert torch.equal(x, y)
        results.append((norm, g))
    assert torch.equal(results[0][0], results[1][0]) and all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))


def test_unaligned_views_and_neighbours(ops):
    """Contiguous views that start off 16 bytes; what lies around them is left as it was."""
    for kind in (F32, BF16):
        buf = tensors([5000], [kind], seed=3)[0]
        keep = buf.clone()
        views = [buf[1:1000], buf[1003:1003 + 2001], buf[4001:4002]]
        n = norm64(views)
        norm = ops.clip_grad_norm_(views, 0.01)
        assert abs(float(norm) - n) <= (U + 1e-12) * n
        mask = torch.ones(5000, dtype=torch.bool, device=DEV)
        for a, b in ((1, 1000), (1003, 3004), (4001, 4002)):
            mask[a:b] = False
        assert torch.equal(buf[mask], keep[mask])
        want = keep[~mask].double() * factor(n, 0.01)
        assert ((buf[~mask].double() - want).abs() <= want.abs() * (2.1 * U + (2.0 ** -8 if kind == BF16 else 0))).all()


def test_large_and_small_magnitudes(ops):
    """Squares beyond fp32's range in both directions."""
    for scale in (1e30, 1e-30):
        g = tensors([1000, 77], [F32, F32], seed=5, scale=scale)
        n = norm64(g)
        norm = ops.clip_grad_norm_(g, float('inf'))
        assert abs(float(norm) - n) <= (U + 1e-12) * n


def test_infinities_and_nan(ops):
    g = tensors([100, 50], [F32, F32], seed=6)
    g[1][3] = float('inf')
    norm = ops.clip_grad_norm_(g, 1.0)
    assert torch.isinf(norm) and not g[0].any() and torch.isnan(g[1][3])  # x * 0, and inf * 0
    g = tensors([100, 50], [F32, BF16], seed=6)
    g[0][3] = float('nan')
    norm = ops.clip_grad_norm_(g, 1.0)
    assert torch.isnan(norm) and all(torch.isnan(x).all() for x in g)


def test_empty_lists(ops, ext):
    for fn in (ops.clip_grad_norm_, ext.clip_grad_norm_):
        assert float(fn([], 1.0)) == 0.0
        assert float(fn([torch.zeros(0, device=DEV)], 1.0)) == 0.0
    for fn in (ops.adamw_clip_step_, ext.adamw_clip_step_):
        assert float(fn([], [], [], [], 1.0, 1e-3, 0.9, 0.999, 1e-6, 0.0)) == 0.0


def adamw64(p, g, m, v, f, lr, b1, b2, eps, wd):
    """Values and bounds of one update from fp32 inputs; constants are taken as the fp32 numbers the kernel gets."""
    r = lambda x: float(torch.tensor(x, dtype=F32))  # noqa: E731
    c1, c2 = r(1 - b1), r(1 - b2)
    lr, b1, b2, eps, wd = map(r, (lr, b1, b2, eps, wd))
    p, g, m, v = (x.cpu().double() for x in (p, g, m, v))
    gg = g * f
    m2, v2 = b1 * m + c1 * gg, b2 * v + c2 * gg * gg
    # f, its product with g, each term and the sum are rounded once each
    em = 4 * U * ((b1 * m).abs() + (c1 * gg).abs()) + 2.0 ** -148
    ev = 6 * U * ((b2 * v).abs() + c2 * gg * gg) + 2.0 ** -148
    root = v2.sqrt() + eps
    upd = m2 / root + wd * p
    # d sqrt(v) = dv / (2 sqrt(v)), and no more than sqrt(dv)
    eroot = torch.minimum(ev / (2 * v2.sqrt().clamp_min(1e-300)), ev.sqrt()) + 2 * U * root
    eu = em / root + m2.abs() * eroot / root ** 2 + 4 * U * (upd.abs() + (wd * p).abs() + (m2 / root).abs())
    return (p - lr * upd, lr * eu + 2 * U * (lr * upd).abs() + U * (p - lr * upd).abs() + U * p.abs()), (m2, em), (v2, ev)


def near(got, want, what):
    val, tol = want
    d = (got.cpu().double() - val).abs()
    assert (d <= tol).all(), (what, float(d.max()), float((d / tol).max()))


@pytest.mark.parametrize('sizes', [[1], [7, 0, 16385], [50001, 3, 400, 20000], [i % 13 + 1 for i in range(130)]])
@pytest.mark.parametrize('max_norm,wd', [(0.01, 0.0), (0.3, 1e-2), (1e9, 1e-5)])
def test_adamw_clip_against_64_bits(ops, ext, sizes, max_norm, wd):
    kinds = [F32] * len(sizes)
    p0, g, m0 = (tensors(sizes, kinds, seed=s) for s in (1, 2, 3))
    v0 = [x.square() for x in tensors(sizes, kinds, seed=4)]
    hyper = (1e-3, 0.9, 0.999, 1e-6, wd)
    n = norm64(g)
    outs = []
    for fn in (ops.adamw_clip_step_, ext.adamw_clip_step_):
        p, m, v = ([x.clone() for x in t] for t in (p0, m0, v0))
        kept = [x.clone() for x in g]
        norm = fn(p, g, m, v, max_norm, *hyper)
        assert abs(float(norm) - n) <= (U + 1e-12) * n
        assert all(torch.equal(a, b) for a, b in zip(g, kept))  # the gradients are left as they are
        outs.append(p + m + v)
        for i in range(len(sizes)):
            wp, wm, wv = adamw64(p0[i], g[i], m0[i], v0[i], factor(n, max_norm), *hyper)
            near(m[i], wm, 'm')
            near(v[i], wv, 'v')
            near(p[i], wp, 'p')
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_adamw_class_with_max_grad_norm(ops):
    """AdamW(max_grad_norm=...) against clipping first and updating with the unclipped class, over three steps: both follow the
    same formula, the clipped gradient rounded to fp32 once more in the second; a parameter without a gradient is left alone."""
    from gzsl_text_amd.modules.common_module import AdamW, clip_grad_norm_
    sizes = [(40, 7), (300,), (3,)]
    gen = torch.Generator().manual_seed(8)
    init = [torch.randn(s, generator=gen) for s in sizes]
    a, b = ([torch.nn.Parameter(x.clone().to(DEV)) for x in init] for _ in range(2))
    oa, ob = AdamW(a, lr=1e-2, weight_decay=1e-3, max_grad_norm=0.5), AdamW(b, lr=1e-2, weight_decay=1e-3)
    for step in range(3):
        for i in (0, 1):
            g = torch.randn(sizes[i], generator=gen).to(DEV)
            a[i].grad, b[i].grad = g.clone(), g.clone()
        oa.step()
        want = norm64([a[0].grad, a[1].grad])
        assert abs(float(oa.grad_norm) - want) <= (U + 1e-12) * want
        clip_grad_norm_(b, 0.5)
        ob.step()
        for x, y in zip(a, b):
            # The unclipped class takes 1 - beta from the rounded beta: 1 - 0.999 is off by half a step of 1, 2^-25 / 1e-3 =
            # 3e-5 of itself, so is v, and half of that sqrt(v); an update is lr * m / sqrt(v) <= 1e-2 * 0.1 / sqrt(1e-3) =
            # 0.032, three of them 0.095 * 1.5e-5 = 1.5e-6.  Roundings besides: ten each of lr * upd, one of p a step.
            assert ((x - y).abs() <= 1.5e-6 + 0.095 * 10 * U + 3 * U * y.abs()).all()
        assert torch.equal(a[2], init[2].to(DEV))
    assert oa.state[a[0]]['step'] == 3 and not oa.state[a[2]]


def test_captured_and_replayed(ops):
    sizes, kinds = [70000, 33, 500], [F32, BF16, F32]
    g = tensors(sizes, kinds, seed=1)
    ops.clip_grad_norm_([x.clone() for x in g], 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm_(g, 0.5)
    for seed in (2, 3, 4):
        new = tensors(sizes, kinds, seed=seed, scale=0.01 * seed)
        for x, y in zip(g, new):
            x.copy_(y)
        graph.replay()
        n2 = ops.clip_grad_norm_(new, 0.5)
        torch.cuda.synchronize()
        assert torch.equal(norm, n2) and all(torch.equal(x, y) for x, y in zip(g, new))
