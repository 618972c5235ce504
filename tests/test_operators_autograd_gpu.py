"""The operators have no autograd function: a call whose result autograd would take for a
constant, or for something else than it is, is refused; an output that a graph has kept is seen
to have changed."""
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError
from operator_refs import Batch

pytestmark = pytest.mark.gpu
A, B = 11, 12


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture
def case():
    b = Batch(51, [6], [0], [4], 16, 24, torch.float32)
    s = psa.Server(0, 1)
    for t, w in ((A, b.a), (B, b.b)):
        s.CreateTable(t, psa.TableInfo(row_capacity=w.shape[1], max_rows=b.rows))
        s.load_rows(t, 0, w.numpy())
    ids = torch.tensor(b.begin, dtype=torch.int32).cuda(), torch.tensor(b.which, dtype=torch.int32).cuda()
    yield b, s, s.create_adapters(A, B, b.adapters()), ids
    s.close()


def _refused(call):
    with pytest.raises(PsxError) as e:
        call()
    assert e.value.status == 1 and "grad" in str(e.value)


def test_adapters_refuse_what_a_graph_would_lose(case):
    b, s, ads, ids = case
    x, base, dy = b.x.cuda(), b.base.cuda(), b.dy.cuda()
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    want, shrunk = ads.forward(x, *ids, base=base)
    dx = torch.zeros_like(x)
    _refused(lambda: ads.forward(leaf(x), *ids, base=base))
    _refused(lambda: ads.forward(x, *ids, base=leaf(base) * 1))   # a clone of it would carry its history
    _refused(lambda: ads.forward(x, *ids, base=base, out=leaf(base)))
    for kw in (dict(x=leaf(x)), dict(dy=leaf(dy)), dict(base=leaf(x)), dict(out=leaf(x))):
        a = dict(dict(x=x, dy=dy, base=x, out=dx), **kw)
        _refused(lambda: ads.backward(a["x"], a["dy"], shrunk, *ids, base=a["base"], out=a["out"]))
    with torch.no_grad():
        assert torch.equal(ads.forward(leaf(x), *ids, base=leaf(base))[0], want)
        ads.backward(leaf(x), leaf(dy), shrunk, *ids, base=leaf(x), out=dx)
    kept = s.checkpoint_store(leaf(x))   # values alone
    assert not kept.load().requires_grad
    _refused(lambda: kept.load(out=leaf(x)))


def test_a_gradient_by_an_autograd_function(case):
    """The way to use them under autograd: the whole of base + adapter, with its gradients."""
    b, s, ads, ids = case

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, base):
            out, shrunk = ads.forward(x, *ids, base=base)
            ctx.save_for_backward(x, shrunk)
            return out

        @staticmethod
        def backward(ctx, dy):
            x, shrunk = ctx.saved_tensors
            dx = torch.zeros_like(x)
            ads.backward(x, dy.contiguous(), shrunk, *ids, out=dx)
            return dx, dy

    x, base = b.x.cuda().requires_grad_(), b.base.cuda().requires_grad_()
    c = b.dy.cuda()
    (Layer.apply(x, base) * c).sum().backward()
    a, w, sc = b.a[b.rows_of(0)].double(), b.b[b.rows_of(0)].double(), b.scales[0]
    want = sc * c.double().cpu() @ w.t() @ a
    mag = sc * c.double().cpu().abs() @ w.abs().t() @ a.abs()
    assert bool(((x.grad.double().cpu() - want).abs() <= (24 + 4 + 16) * 2.0 ** -23 * mag).all())
    assert torch.equal(base.grad, c)


def test_outputs_that_a_graph_has_kept(case):
    b, s, ads, ids = case
    x, base = b.x.cuda(), b.base.cuda()

    def kept(out, write):
        w = torch.ones_like(out, requires_grad=True)
        y = (w * out).sum()   # keeps out
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()

    out, shrunk = ads.forward(x, *ids, base=base)
    kept(out, lambda: ads.forward(x, *ids, base=base, out=out))
    dx = torch.zeros_like(x)
    ga, gb = ads.backward(x, b.dy.cuda(), shrunk, *ids, out=dx)
    for t in (dx, ga, gb):
        kept(t, lambda: ads.backward(x, b.dy.cuda(), shrunk, *ids, out=dx, grad_a=ga, grad_b=gb))
    z = s.checkpoint_store(x)
    kept(dx, lambda: z.load(out=dx))
    with torch.inference_mode():
        y = torch.zeros_like(base)
        ads.forward(x, *ids, base=base, out=y)


def test_position_bias(case):
    b, s, ads, ids = case
    s.CreateTable(7, psa.TableInfo(row_capacity=3, max_rows=8))
    bias = s.position_bias(7, 0, 8, 16, True)
    out, d = torch.zeros(3, 4, 5, device="cuda"), torch.ones(1, 3, 4, 5, device="cuda")
    _refused(lambda: bias.forward(4, 5, out=out.clone().requires_grad_()))
    _refused(lambda: bias.backward(d.clone().requires_grad_()))
    w = torch.ones_like(out, requires_grad=True)
    y = (w * out).sum()
    bias.forward(4, 5, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    grad = bias.backward(d)
    w = torch.ones_like(grad, requires_grad=True)
    y = (w * grad).sum()
    bias.backward(d, grad=grad)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_forward_pass_over_a_buffer_that_another_keeps(case):
    """Two passes that keep one shrunk buffer for their gradients: the first's is gone, and said so."""
    b, s, ads, ids = case
    buffer = torch.empty(ads.sizes(b.T)[0] // 4, device="cuda")

    class Layer(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, shrunk):
            out, shrunk = ads.forward(x, *ids, shrunk=shrunk)
            ctx.save_for_backward(x, shrunk)
            return out

        @staticmethod
        def backward(ctx, dy):
            x, shrunk = ctx.saved_tensors
            dx = torch.zeros_like(x)
            ads.backward(x, dy.contiguous(), shrunk, *ids, out=dx)
            return dx, None

    x = b.x.cuda().requires_grad_()
    first = Layer.apply(x, buffer)
    second = Layer.apply(2 * x, buffer)
    second.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        first.sum().backward()
