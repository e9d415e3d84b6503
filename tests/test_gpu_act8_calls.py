"""GPU tests of calls of the 8-bit checkpoint operators at the edges of what they accept."""
import numpy as np
import pytest
import torch

import test_gpu_act8 as base
from oracle import act8 as oa

pytestmark = pytest.mark.gpu
SLOPE = base.SLOPE


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
