"""CPU tests of what the entry points of the 8-bit checkpoint operators refuse."""
import pytest
import torch

from deepwmh_amd import act8


def _ck(shape, fmt='e4m3'):
    return act8.Act8.empty(shape, fmt, 'cpu')


def test_a_tensor_that_requires_grad_is_refused():
    """The calls record nothing for autograd: their results would silently have no gradient."""
    new = lambda *s: torch.zeros(s, requires_grad=True)         # noqa: E731
    x, st, ck = torch.zeros(1, 2, 5), torch.zeros(1, 2, 2), _ck((1, 2, 5))
    bwd = lambda **kw: act8.instnorm_lrelu_backward(ck, *(kw.pop(n, st) for n in ('ss', 'mr')), **dict(dict(g1=x), **kw))      # noqa: E731
    calls = [lambda: act8.pack(new(1, 2, 5)), lambda: act8.pack(x, ss=new(1, 2, 2)), lambda: act8.pack_columns(new(1, 2, 5)),
             lambda: act8.pack(new(1, 2, 10)[..., ::2]), lambda: act8.pack(new(2, 5)[None] * 2), lambda: act8.unpack(ck, ss=new(1, 2, 2)),
             lambda: act8.unpack(ck, out=new(1, 2, 5)), lambda: act8.product(ck, _ck((1, 3, 5)), out=new(1, 2, 3)),
             lambda: bwd(ss=new(1, 2, 2)), lambda: bwd(mr=new(1, 2, 2)), lambda: bwd(gamma=torch.nn.Parameter(torch.ones(2))), lambda: bwd(g1=new(1, 2, 5)),
             lambda: bwd(g2=new(1, 2, 5)), lambda: bwd(dlogits=new(1, 3, 5), wseg=torch.zeros(3, 2)), lambda: bwd(dlogits=torch.zeros(1, 3, 5), wseg=new(3, 2)),
             lambda: act8.convtranspose_weight_gradient(new(1, 2, 2, 2, 2), None, torch.zeros(1, 3, 2, 4, 4)),
             lambda: act8.convtranspose_weight_gradient(torch.zeros(1, 2, 2, 2, 2), None, new(1, 3, 2, 4, 4)),
             lambda: act8.convtranspose_weight_gradient(torch.zeros(1, 2, 2, 2, 2), new(1, 2, 2), torch.zeros(1, 3, 2, 4, 4))]
    for k, call in enumerate(calls):
        with pytest.raises(RuntimeError, match='requires grad'):
            call()
            pytest.fail('call %d was taken' % k)
        with torch.no_grad(), pytest.raises(RuntimeError, match='no CPU path'):
            call()
            pytest.fail('call %d was taken' % k)


def test_shapes_that_are_no_checkpoints_are_refused():
    for shape in ((2, 3), (1, 2, -5), ()):
        with pytest.raises(ValueError, match='expected'):
            act8.Act8.empty(shape, 'int8', 'cpu')
    st = torch.zeros(1, 1, 2)
    with pytest.raises(ValueError, match='wseg'):               # (a number is no [K, C])
        act8.instnorm_lrelu_backward(_ck((1, 1, 5)), st, st, dlogits=torch.zeros(1, 1, 5), wseg=torch.tensor(1.0))
