"""Gradients through rotary: against the formula's in 64 bits and against differences of results."""

import pytest
import torch

import quashkv_amd as Q
from quashkv_amd import _native as N
from quashkv_amd.rotary import rotary
from tests import shared_reference as S

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a HIP device")
    N.lib()


def _rows(rows, heads, d, dtype, seed):
    return torch.randn(rows, heads, d, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _turns(R):
    return Q.rotary_turns(Q.rotary_frequencies(R), DEV)


def _near(got, g, pos, turns, factor, pairs, inverse=True):
    y, tol = S.turned(g.cpu(), pos.tolist(), turns.tolist(), factor, pairs, inverse)
    assert got.dtype is g.dtype
    assert ((got.cpu().double() - y).abs() <= tol + HALF[g.dtype] * (y.abs() + tol)).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,Hq,Hk,d,R,pairs,factor", [
    (1, 1, 1, 8, 8, False, 1.0), (37, 8, 2, 64, 64, False, 1.25), (5, 3, 3, 96, 40, True, 0.8),
    (130, 4, 1, 70, 34, False, 1.0), (1, 5, 2, 7, 6, True, 2.0)])
def test_gradient_is_the_formulas(rows, Hq, Hk, d, R, pairs, factor, dtype):
    pos = torch.randint(-5, 1 << 20, (rows,), generator=torch.Generator().manual_seed(3)).int().to(DEV)
    turns = _turns(R)
    for inverse in (False, True):
        q, k = _rows(rows, Hq, d, dtype, 1).requires_grad_(), _rows(rows, Hk, d, dtype, 2).requires_grad_()
        a, b = rotary(q, k, pos, turns, factor, interleaved=pairs, inverse=inverse)
        with torch.no_grad():
            x, y = rotary(q, k, pos, turns, factor, interleaved=pairs, inverse=inverse)
        assert torch.equal(a, x) and torch.equal(b, y) and not x.requires_grad
        g, h = _rows(rows, Hq, d, dtype, 4), _rows(rows, Hk, d, dtype, 5)
        torch.autograd.backward((a, b), (g, h))
        _near(q.grad, g, pos, turns, factor, pairs, not inverse)
        _near(k.grad, h, pos, turns, factor, pairs, not inverse)


def test_differences():
    """The map is linear: sum g (f(x + e) - f(x)) = sum e grad, each result within its bound."""
    pos, turns = torch.arange(1000, 1020, dtype=torch.int32, device=DEV), _turns(48)
    x, e, g = (_rows(20, 3, 64, F32, s) for s in (1, 2, 3))
    for pairs in (False, True):
        t = x.clone().requires_grad_()
        a, _ = rotary(t, None, pos, turns, 0.8, interleaved=pairs)
        a.backward(g)
        f = [rotary(z.cpu().to(DEV), None, pos, turns, 0.8, interleaved=pairs)[0].double() for z in (x + e, x)]
        z = (x + e).double() - x.double()                 # (what the sum is, rounded)
        left = (g.double() * (f[0] - f[1])).sum()
        right = (z * t.grad.double()).sum()
        tol = 0.0
        for v, w, inv in ((x + e, g, False), (x, g, False), (g, z, True)):
            y, off = S.turned(v.cpu(), pos.tolist(), turns.tolist(), 0.8, pairs, inv)
            tol += float((w.cpu().double().abs() * (off + HALF[F32] * (y.abs() + off))).sum())
        assert abs(float(left - right)) <= tol


def test_who_gets_a_gradient():
    pos, turns = torch.arange(6, dtype=torch.int32, device=DEV), _turns(16)
    make = lambda h, s: _rows(6, h, 16, F32, s)
    # keys alone, queries alone, no keys, a result that the loss does not ask for
    q, k = make(4, 1), make(2, 2).requires_grad_()
    a, b = rotary(q, k, pos, turns)
    b.backward(make(2, 3))
    _near(k.grad, make(2, 3), pos, turns, 1.0, False)
    assert q.grad is None
    q, k = make(4, 1).requires_grad_(), make(2, 2)
    a, b = rotary(q, k, pos, turns)
    a.backward(make(4, 3))
    _near(q.grad, make(4, 3), pos, turns, 1.0, False)
    q = make(4, 1).requires_grad_()
    a, none = rotary(q, None, pos, turns)
    assert none is None
    a.backward(make(4, 3))
    _near(q.grad, make(4, 3), pos, turns, 1.0, False)
    q, k = make(4, 1).requires_grad_(), make(2, 2).requires_grad_()
    a, b = rotary(q, k, pos, turns)
    b.backward(make(2, 3))
    assert q.grad is None and k.grad is not None


def test_broadcast_rows_heads_and_gradients():
    """Rows of one, heads of one, and a gradient that is a number, broadcast."""
    pos, turns = torch.arange(6, dtype=torch.int32, device=DEV), _turns(16)
    one = _rows(1, 1, 16, F32, 1).requires_grad_()
    a, b = rotary(one.expand(6, 4, 16), one.expand(6, 1, 16), pos, turns)
    (a.sum() + 2 * b.sum()).backward()
    y, tol = S.turned(torch.ones(6, 1, 16), pos.tolist(), turns.tolist(), 1.0, False, True)
    # four heads of weight 1 and one of 2, 24 sums of rounded gradients of up to 1.5
    want, off = 6 * y.sum((0, 1)), 6 * tol.sum((0, 1)) + 30 * 24 * 1.5 * 2.0 ** -24
    assert ((one.grad.flatten().cpu().double() - want).abs() <= off).all()


def test_positions_of_the_step_that_ran():
    """A plan's positions move on between a call and its backward pass."""
    pos, turns = torch.arange(6, dtype=torch.int32, device=DEV), _turns(16)
    was = pos.clone()
    q = _rows(6, 2, 16, F32, 1).requires_grad_()
    a, _ = rotary(q, None, pos, turns)
    pos.data.add_(100)
    a.backward(_rows(6, 2, 16, F32, 2))
    _near(q.grad, _rows(6, 2, 16, F32, 2), was, turns, 1.0, False)


def test_second_derivatives_and_empty_rows():
    pos, turns = torch.arange(6, dtype=torch.int32, device=DEV), _turns(16)
    q, g = _rows(6, 2, 16, F32, 1).requires_grad_(), _rows(6, 2, 16, F32, 2).requires_grad_()
    a, _ = rotary(q, None, pos, turns)
    d, = torch.autograd.grad(a, q, g, create_graph=True)
    h = _rows(6, 2, 16, F32, 3)
    e, = torch.autograd.grad(d, g, h)               # the map itself
    _near(e, h, pos, turns, 1.0, False, False)
    z = torch.zeros(0, 2, 16, device=DEV, requires_grad=True)
    a, _ = rotary(z, None, pos[:0], turns)
    a.sum().backward()
    assert z.grad.shape == (0, 2, 16)


def test_on_another_stream():
    pos, turns = torch.arange(64, dtype=torch.int32, device=DEV), _turns(16)
    q, g = _rows(64, 2, 16, F32, 1).requires_grad_(), _rows(64, 2, 16, F32, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, _ = rotary(q, None, pos, turns)
        a.backward(g)
    torch.cuda.current_stream().wait_stream(s)
    _near(q.grad, g, pos, turns, 1.0, False)


def test_given_outputs_take_no_gradients():
    pos, turns = torch.arange(6, dtype=torch.int32, device=DEV), _turns(16)
    q, k = _rows(6, 2, 16, F32, 1), _rows(6, 2, 16, F32, 2)
    w = q.clone().requires_grad_()
    for args in (dict(q=w, k=None, q_out=torch.empty_like(q)), dict(q=w * 1, k=k, k_out=k),
                 dict(q=q, k=w, q_out=q), dict(q=q, k=None, q_out=w)):
        with pytest.raises(ValueError, match="gradient"):
            rotary(**args, positions=pos, turns=turns)
    x = (w * 1)
    with torch.no_grad():
        rotary(x, None, pos, turns, q_out=x)
    assert torch.equal(x, rotary(q, None, pos, turns)[0])


def test_captured():
    """A call and its gradient in a graph, replayed against eager ones, with other positions each time."""
    turns = _turns(48)
    pos = torch.zeros(40, dtype=torch.int32, device=DEV)
    q, k = _rows(40, 4, 64, BF16, 1).requires_grad_(), _rows(40, 2, 64, BF16, 2).requires_grad_()
    g, h = _rows(40, 4, 64, BF16, 3), _rows(40, 2, 64, BF16, 4)

    def step():
        a, b = rotary(q, k, pos, turns, 1.5)
        return (a.detach(), b.detach()) + torch.autograd.grad((a, b), (q, k), (g, h))

    step()                                  # (what a first call sets up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        pos.copy_(torch.arange(40) * (i + 1))
        with torch.no_grad():
            q.copy_(_rows(40, 4, 64, BF16, 10 + i))
        g.copy_(_rows(40, 4, 64, BF16, 20 + i))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i
