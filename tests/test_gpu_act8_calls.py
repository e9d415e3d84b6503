"""GPU tests of calls of the 8-bit checkpoint operators at the edges of what they accept: sizes of a real training step, infinite gradients, scales at
both ends of the range, batches of many small products."""
import math

import numpy as np
import pytest
import torch

import test_gpu_act8 as base
import test_gpu_act8_trainer as steps
from oracle import act8 as oa

pytestmark = pytest.mark.gpu
U, HALF, SLOPE = base.U, base.HALF, base.SLOPE


# ---- a head whose logit gradient is not finite ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize('shape', [(1, 3, 500), (2, 5, 3, 7, 11), (2, 3, 8193), (9, 2, 302)], ids=lambda s: 'x'.join(map(str, s)))
@pytest.mark.parametrize('K', [1, 2, 3, 4])
def test_backward_of_an_infinite_logit_gradient(K, shape):
    """dA = wseg^T dl takes its infinity from the classes that there are: a sum with one infinity in it is that infinity, not NaN."""
    from deepwmh_amd import act8
    rng = np.random.default_rng(30)
    N, C = shape[:2]
    S = int(np.prod(shape[2:]))
    y0 = rng.standard_normal((N, C, S)).astype(np.float32)
    ss, mr, gamma = base._norm_of(y0.astype(np.float64), rng)
    y = oa.values(*oa.quantise(y0, 'int8'), S)
    wseg = rng.standard_normal((K, C)).astype(np.float32)
    dev = lambda a, sh=None: torch.from_numpy(a).view(sh if sh else a.shape).cuda()            # noqa: E731
    ck = act8.pack(dev(y0, shape), 'int8')
    for k in range(K):
        dl = rng.standard_normal((N, K, S)).astype(np.float32)
        dl[0, k, S // 3] = np.inf
        got = act8.instnorm_lrelu_backward(ck, dev(ss), dev(mr), dev(gamma), dlogits=dev(dl, (N, K) + shape[2:]), wseg=dev(wseg), slope=SLOPE)
        with np.errstate(invalid='ignore'):
            want, _ = oa.instnorm_lrelu_backward(y, ss, mr, gamma.astype(np.float64), None, None, dl.astype(np.float64), wseg.astype(np.float64),
                                                 float(np.float32(SLOPE)))
        assert np.isinf(want['dbeta']).all() and np.isinf(want['dgamma']).all()
        for name in ('dbeta', 'dgamma', 'dwseg'):
            g, w = base._np(getattr(got, name)), want[name]
            off = ~np.isfinite(w)
            assert np.array_equal(np.isfinite(g), ~off) and np.array_equal(g[off], w[off]), (name, k)
        dy = base._np(got.dy).reshape(N, C, S)
        assert not np.isfinite(dy[0]).any() and np.isfinite(dy[1:]).all()


# ---- products ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dims', [(1, 300, 520, 200), (3, 61, 136, 1000), (1, 512, 512, 1024), (1, 1030, 4100, 520), (1, 3590, 3601, 4480), (1, 64, 256, 40000)],
                         ids=lambda d: 'x'.join(map(str, d)))
def test_bfloat16_product_is_off_by_its_results_rounding(dims):
    """Of random terms.  A result's rounding to bfloat16 is uniform over a step of at most 2^-7 of it: 2^-7 / sqrt(12) = 2.26e-3 in the norm at most.
    In front of it eight products lose up to seven terms' bits below 2^-13 of the largest, toward zero, which for products of normal variables (the
    largest of eight: 2.5) is 2.5 2^-13 sqrt(7 / 3) of the sum's own sqrt(8): 1.7e-4.  Together 2.27e-3."""
    from deepwmh_amd import act8
    B, M, N, K = dims
    g = torch.Generator(device='cuda').manual_seed(31)
    a, b = (act8.pack(torch.randn(B, r, K, device='cuda', generator=g), 'e4m3') for r in (M, N))
    c = torch.matmul(act8.unpack(a).double(), act8.unpack(b).double().transpose(1, 2).contiguous())
    for total in (False, True):
        want = c.sum(0) if total else c
        got = act8.product(a, b, dtype=torch.bfloat16, sum_batches=total).double()
        assert float((got - want).norm() / want.norm()) <= 2.3e-3


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('dims', [(40, 35, 300), (20, 40, 300), (300, 70, 9000), (1100, 4200, 130), (3500, 3600, 260), (3500, 3600, 4200)],
                         ids=lambda d: 'x'.join(map(str, d)))
def test_products_of_scales_over_the_whole_range(dims, dtype):
    """Rows of a and b with exponent bytes from the smallest to nearly the largest, so that a product of blocks lies anywhere between 2^-250 and 2^240."""
    from deepwmh_amd import act8
    M, N, K = dims
    g = torch.Generator(device='cuda').manual_seed(32)
    a, b = (torch.randn(1, r, K, device='cuda', generator=g, dtype=torch.float64) for r in (M, N))
    for t in (a, b):
        e = torch.randint(-124, 125, (1, t.shape[1], -(-K // 128)), device='cuda', generator=g).double()
        e[:, ::2] = e[:, ::2, :1]                               # every second row of one size, the others with blocks of any
        t *= torch.exp2(e).repeat_interleave(128, -1)[..., :K]
    a, b = (act8.pack(t.float().clamp(-2.0 ** 127, 2.0 ** 127), 'e4m3') for t in (a, b))
    assert int(a.scales[..., :-(-K // 128)].min()) <= 2 and int(a.scales.max()) >= 240
    va, vb = act8.unpack(a).double(), act8.unpack(b).double()
    c, mag = (torch.matmul(x, y.transpose(1, 2).contiguous())[0] for x, y in ((va, vb), (va.abs(), vb.abs())))
    got = act8.product(a, b, dtype=dtype)[0].double()
    # as for ordinary sizes; and a number below 2^-126, a product of two codes or a sum that is joined or stored, may be lost
    tol = min(-(-K // 128) * 2 + 64, 600) * 2.0 ** -23 * mag + HALF[dtype] * c.abs() + (K + 300) * 2.0 ** -126
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -10 * mag
    else:                                                       # codes widened with their scale are bfloat16 numbers: so may one of them below 2^-126
        la, lb = (t.abs() * (t.abs() < 2.0 ** -126) for t in (va, vb))
        tol = tol + torch.matmul(la, vb.abs().transpose(1, 2).contiguous())[0] + torch.matmul(va.abs(), lb.transpose(1, 2).contiguous())[0]
    fits, over = mag < 2.0 ** 127, c.abs() >= 2.0 ** 129
    assert int(fits.sum()) > M * N // 8 and not bool(torch.isfinite(got[over]).any())
    assert bool(torch.isfinite(got[fits]).all()) and bool(((got - c).abs() <= tol)[fits].all())
    small = fits & (c.abs() > 2.0 ** -100) & (mag < 2.0 ** 100) & (c.abs() > mag / 16)
    assert int(small.sum()) > M * N // 64 and bool((got[small] != 0).all())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('dims', [(256, 64, 64, 512), (200, 40, 200, 700), (192, 33, 33, 130), (211, 61, 136, 1000), (6, 40, 8192, 260), (300, 33, 257, 129), (64, 128, 96, 2048)],
                         ids=lambda d: 'x'.join(map(str, d)))
def test_products_of_many_small_items(dims, dtype):
    base.test_product_of_larger_odd_sizes(dims, dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_product_gives_the_same_bits_between_other_work(dtype):
    from deepwmh_amd import act8
    g = torch.Generator(device='cuda').manual_seed(33)
    sets = [tuple(act8.pack(torch.randn(B, r, K, device='cuda', generator=g), 'e4m3') for r in (M, N)) for B, M, N, K in ((3, 61, 136, 1000), (1, 300, 500, 3000), (2, 17, 90, 9000))]
    want = [act8.product(a, b, dtype=dtype) for a, b in sets]
    for k in range(30):
        for i in (0, 1, 2) if k % 2 else (2, 0, 1):
            assert torch.equal(act8.product(*sets[i], dtype=dtype), want[i])


# ---- tensors of a real step ----------------------------------------------------------------------------------------------------------------
LONG = 127 * 129 * 131                                          # an odd row of 2.1 million; 24 of them are past the 192 MB where accesses pass the caches


def _quantise(z, fmt):
    """float64 [R, L] finite -> code values [R, L], exponents [R, blocks] (written for the GPU, from the definition)."""
    R, L = z.shape
    nb = -(-L // 128)
    z = torch.nn.functional.pad(z, (0, nb * 128 - L)).view(R, nb, 128)
    top = 127.0 if fmt == 'int8' else 448.0
    high = z.abs().amax(-1)
    m, k = torch.frexp(high / top)
    e = torch.where(high == 0, -126, torch.where(m == 0.5, k - 1, k).clamp(min=-126))
    q = z / torch.exp2(e.double())[..., None]
    if fmt == 'int8':
        codes = q.round()
    else:
        step = torch.exp2((torch.frexp(q).exponent - 1).clamp(min=-6).double() - 3)
        codes = (q / step).round() * step
    return codes.view(R, -1)[:, :L], e


def _values(codes, e):
    return codes * torch.exp2(e.double()).repeat_interleave(128, -1)[:, :codes.shape[1]]


def _grid(fmt):
    if fmt == 'int8':
        return torch.arange(-127, 128, device='cuda', dtype=torch.float64)
    m = torch.arange(127, dtype=torch.float64)
    mag = torch.where(m < 8, m * 2.0 ** -9, (8 + m % 8) * torch.exp2(torch.floor(m / 8) - 10))
    return torch.cat([-mag.flip(0)[:-1], mag]).cuda()


def _kept(z, codes, e, sc, sh, fmt):
    """codes with those on the wrong side of z sc + sh = 0 moved to the neighbour on z's."""
    grid = _grid(fmt)
    v = _values(codes, e)
    want, got = z * sc + sh > 0, v * sc + sh > 0
    at = torch.searchsorted(grid, codes.contiguous())
    moved = grid[(at + torch.where(want == (sc > 0), 1, -1)).clamp(0, grid.numel() - 1)]
    return torch.where(want != got, moved, codes)


def _long(C, g, dtype=torch.float32):
    x = torch.randn(1, C, LONG, device='cuda', generator=g)
    x *= torch.exp(torch.randn(1, C, 1, device='cuda', generator=g))
    x += torch.randn(1, C, 1, device='cuda', generator=g)
    ss = torch.stack([1 + 0.3 * torch.randn(1, C, device='cuda', generator=g), torch.randn(1, C, device='cuda', generator=g)], -1)
    return x.to(dtype), ss


@pytest.mark.parametrize('mode', ['plain', 'activate', 'keep_sign'])
@pytest.mark.parametrize('fmt', ['int8', 'e4m3'])
@pytest.mark.parametrize('dtype,C', [(torch.float32, 24), (torch.bfloat16, 48)])
def test_pack_and_unpack_past_the_caches(dtype, C, fmt, mode):
    from deepwmh_amd import act8
    x, ss = _long(C, torch.Generator(device='cuda').manual_seed(34), dtype)
    assert x.numel() * x.element_size() > 192 << 20
    ck = act8.pack(x, fmt, ss=None if mode == 'plain' else ss, slope=SLOPE, keep_sign=mode == 'keep_sign')
    nb = -(-LONG // 128)
    backs = [act8.unpack(ck, dtype), act8.unpack(ck, dtype, ss=ss, slope=SLOPE)]
    assert not bool(ck.codes[..., LONG:].float().any()) and not bool(ck.scales[..., nb:].any())
    slope = torch.tensor(SLOPE, device='cuda')
    for c in range(C):
        z, sc, sh = x[0, c].double()[None], ss[0, c, 0].double(), ss[0, c, 1].double()
        if mode == 'activate':
            z = (z * sc + sh).float()                           # (a float64 product of two float32 is exact)
            z = torch.where(z > 0, z, z * slope).double()
        codes, e = _quantise(z, fmt)
        if mode == 'keep_sign':
            codes = _kept(z, codes, e, sc, sh, fmt)
        assert torch.equal(ck.codes[0, c, :LONG].double()[None], codes) and torch.equal(ck.scales[0, c, :nb].int() - 127, e[0].int()), c
        v = _values(codes, e)[0]
        a = (v * sc + sh).float()
        a = torch.where(a > 0, a, a * slope).double()
        assert torch.equal(backs[0][0, c], v.to(dtype))
        # the activation is rounded as it is formed (a second time where it is negative, by the slope) and to its type
        assert bool(((backs[1][0, c].double() - a).abs() <= (HALF[dtype] + 2 * U) * a.abs() + 2.0 ** -140).all()), c


@pytest.mark.parametrize('K,use2', [(0, False), (2, False), (3, True)])
@pytest.mark.parametrize('fmt', ['int8', 'e4m3'])
def test_backward_past_the_caches(fmt, K, use2):
    """Rows of which the first ones are read past the caches, and the last ones not; tolerances as for short rows (test_gpu_act8)."""
    from deepwmh_amd import act8
    C = 40
    g = torch.Generator(device='cuda').manual_seed(35)
    x, _ = _long(C, g)
    ck = act8.pack(x, fmt)
    mean, rstd = x.double().mean(-1), 1 / (x.double().var(-1, unbiased=False) + 1e-5).sqrt()
    gamma, beta = 1 + 0.2 * torch.randn(C, device='cuda', generator=g), 0.2 * torch.randn(C, device='cuda', generator=g)
    mr = torch.stack([mean, rstd], -1).float()
    ss = torch.stack([gamma * rstd, beta - mean * gamma * rstd], -1).float()
    new = lambda *s: 1e-2 * torch.randn(s, device='cuda', generator=g)           # noqa: E731
    g1, g2, dl, wseg = new(1, C, LONG), new(1, C, LONG) if use2 else None, new(1, K, LONG) if K else None, new(K, C) if K else None
    assert C * LONG * (9 if use2 else 5) > 256 << 20
    got = act8.instnorm_lrelu_backward(ck, ss, mr, gamma, g1=g1, g2=g2, dlogits=dl, wseg=wseg, slope=SLOPE)
    y32 = act8.unpack(ck)
    slope = float(np.float32(SLOPE))
    for c in range(C):
        y, sc, sh = y32[0, c].double(), ss[0, c, 0].double(), ss[0, c, 1].double()
        z = y * sc + sh
        terms = [t[0, c].double() for t in (g1, g2) if t is not None] + [wseg[k, c].double() * dl[0, k].double() for k in range(K)]
        d = torch.where(z > 0, 1.0, slope)
        dz, mag = sum(terms) * d, sum(t.abs() for t in terms) * d
        xh = (y - mr[0, c, 0].double()) * mr[0, c, 1].double()
        gr = gamma[c].double() * mr[0, c, 1].double()
        dy = gr * (dz - dz.mean() - xh * (dz * xh).mean())
        tol = 16 * U * gr.abs() * (mag + mag.mean() + xh.abs() * (mag * xh.abs()).mean()) + 2.0 ** -140
        assert bool(((got.dy[0, c].double() - dy).abs() <= tol).all()), c
        pairs = [(got.dbeta[c], dz.sum(), mag.sum()), (got.dgamma[c], (dz * xh).sum(), (mag * xh.abs()).sum()), (got.dbias[c], dy.sum(), tol.sum() / (16 * U))]
        for k in range(K):
            t = dl[0, k].double()
            pairs.append((got.dwseg[k, c], (z * d * t).sum(), (t.abs() * ((z * d).abs() + sh.abs() + (y * sc).abs())).sum()))
        for have, want, size in pairs:
            assert abs(float(have) - float(want)) <= 16 * U * float(size) + 2.0 ** -140, c


# ---- a training step -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('kind', ['tiny', 'aniso', 'wide'])
@pytest.mark.parametrize('fmt,most', [('int8', 0.05), ('e4m3', 0.13)])
def test_every_gradient_of_a_checkpointed_step_is_finite(kind, fmt, most, tiny_net):
    """And near the exact one (bounds of test_gpu_act8_trainer).  Only a gradient that is identically zero has no relative error: a head whose weight in
    the loss is zero, where the checkpointed one is zero too."""
    from deepwmh_amd.trainer import UNetTrainer
    plan, sd, x, lab = steps._setup(kind, tiny_net)
    td = steps._targets(plan, lab)
    plain, tr = UNetTrainer(plan, sd, 'cuda:0'), UNetTrainer(plan, sd, 'cuda:0', checkpoint8=fmt)
    for t in (plain, tr):
        t.forward(x)
        t.backward(td)
    a, b = steps._grads(plain), steps._grads(tr)
    measured = 0
    for n in a:
        assert np.isfinite(a[n]).all() and np.isfinite(b[n]).all(), n
        if not a[n].any():
            assert not b[n].any(), n
        elif kind == 'wide' and (n.endswith('conv.weight') or 'tu' in n or 'seg' in n):
            measured += 1
            assert math.isfinite(np.linalg.norm(b[n])) and np.linalg.norm(a[n] - b[n]) <= most * np.linalg.norm(a[n]), n
    assert measured > 10 or kind != 'wide'
