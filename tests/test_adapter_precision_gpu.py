"""How far the adapters' products of bf16 parts may be off a single product, where every bit of a
mantissa counts: one rank, one product a value, and a base that cancels it.

A part is the nearest bf16 to what the parts before it left, so 2^-8 of a value at most is left
behind the first and 2^-17 behind the second.  Two parts a factor (16-bit outputs) leave out the
product of the second parts, 2^-16 at most, and each factor's 2^-17: 2^-15 of the product.  The
tolerance of operator_refs.Batch is that, the f32 additions and the output's rounding."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from operator_refs import Batch, off

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]
A, B = 11, 12
# next to the borders at which a first or a second part rounds the other way or is farthest off
EDGES = [1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -23,
         1 + 2.0 ** -8 - 2.0 ** -17 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -17 - 2.0 ** -23, 1 + 2.0 ** -7 + 2.0 ** -16,
         1 + 2.0 ** -8 - 2.0 ** -16, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 2 - 2.0 ** -23, 1.0]


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _set(b):
    s = psa.Server(0, 1)
    for t, w in ((A, b.a), (B, b.b)):
        s.CreateTable(t, psa.TableInfo(row_capacity=w.shape[1], max_rows=b.rows))
        s.load_rows(t, 0, w.numpy())
    return s, s.create_adapters(A, B, b.adapters()), torch.tensor(b.begin, dtype=torch.int32).cuda(), \
        torch.tensor(b.which, dtype=torch.int32).cuda()


def _check(b):
    s, ads, begin, which = _set(b)
    out, shrunk = ads.forward(b.x.cuda(), begin, which, base=b.base.cuda())
    want, tol = b.forward(torch.zeros(b.T, b.d_out))
    assert off(out, want, tol) <= 1
    dx = torch.zeros(b.T, b.d_in, dtype=b.dtype, device="cuda")
    ga, gb = ads.backward(b.x.cuda(), b.dy.cuda(), shrunk, begin, which, base=b.dbase.cuda(), out=dx)
    want, tol = b.backward(torch.zeros(b.T, b.d_in), 1.0)
    for name, g in (("dx", dx), ("grad_a", ga), ("grad_b", gb)):
        assert off(g, want[name], tol[name]) <= 1, name
    s.sync()
    s.close()


def _mantissas(n):
    r = np.random.RandomState(3).uniform(1, 2, size=n).astype(np.float32)
    return torch.from_numpy(np.concatenate([np.array(EDGES, np.float32), r]))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("sign", [1, -1])
def test_forward_products_of_edge_mantissas(dt, sign):
    """v = A of one token times each B; the base takes the product away."""
    m = _mantissas(53)
    n = len(m)
    b = Batch(1, [1] * n, list(range(n)), [1] * n, 1, n, dt, scales=[1.0] * n)
    b.x = torch.full((n, 1), float(sign)).to(dt)
    b.a[b.first] = m[:, None]
    b.b[b.first] = m
    b.base = (-sign * m.double()[:, None] * m.double()).to(dt)
    _check(b)


@pytest.mark.parametrize("dt", DT)
def test_backward_products_of_edge_mantissas(dt):
    """u = B of one token's dy times each A; the base of dx takes the product away."""
    m = _mantissas(53)
    n = len(m)
    b = Batch(2, [1] * n, list(range(n)), [1] * n, n, 1, dt, scales=[1.0] * n)
    b.dy = torch.ones(n, 1).to(dt)
    b.b[b.first] = m[:, None]
    b.a[b.first] = m
    b.dbase = (-m.double()[:, None] * m.double()).to(dt)
    _check(b)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_rounding_has_no_direction(dt):
    """4096 products of two drawn mantissas in [0.5, 1), base taken away: parts that always fall
    short are short by 2^-16 of the sum or more.  Independent errors of either sign, 2^-15 at most
    each, add to more than 8 sqrt(4096) 2^-15 with a chance below 2 exp(-32); the outputs, at most
    2^-9, are rounded by 2^-18 at most."""
    n = 4096
    r = np.random.RandomState(5).uniform(0.5, 1, size=(2, n, 1)).astype(np.float32)
    b = Batch(3, [1] * n, list(range(n)), [1] * n, 1, 1, dt, scales=[1.0] * n)
    b.x = torch.ones(n, 1).to(dt)
    b.a[b.first], b.b[b.first] = torch.from_numpy(r[0]), torch.from_numpy(r[1])
    prod = torch.from_numpy(r[0].astype(np.float64) * r[1])
    b.base = (-prod).to(dt)
    s, ads, begin, which = _set(b)
    out = ads.forward(b.x.cuda(), begin, which, base=b.base.cuda())[0].cpu().double()
    assert abs(float((out - prod - b.base.double()).sum())) <= 8 * 64 * (2.0 ** -15 + 2.0 ** -18)
    s.close()


@pytest.mark.parametrize("dt", DT)
def test_finite_values_next_to_the_largest(dt):
    """A factor past the largest bf16 is no infinity: rows, activations, and what lies between."""
    top = torch.finfo(torch.float32).max
    edge = 3.3961775e38   # from here on the nearest bf16 is an Inf
    n = 5
    b = Batch(4, [1] * n, list(range(n)), [1] * n, 1, n, dt, scales=[1e-6] * n)
    one = torch.ones(n, 1)
    for big in (top, -top, edge, 3.39e38):
        b.x, b.base, b.dbase = one.to(dt), torch.zeros(n, n).to(dt), torch.zeros(n, 1).to(dt)
        b.dy = torch.full((n, n), 2.0 ** -6).to(dt)
        b.a[b.first] = big          # v itself is large
        b.b[b.first] = 1e-31
        _check_forward(b)
        b.a[b.first] = 1e-31
        b.b[b.first] = big
        _check(b)
        if dt == torch.float32:
            b.x = one * big
            b.b[b.first] = 1.0
            _check(b)


def _check_forward(b):
    s, ads, begin, which = _set(b)
    out = ads.forward(b.x.cuda(), begin, which, base=b.base.cuda())[0]
    want, tol = b.forward(torch.zeros(b.T, b.d_out))
    assert off(out, want, tol) <= 1
    s.close()
