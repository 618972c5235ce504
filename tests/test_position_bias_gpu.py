"""The relative position bias whose buckets are rows of a table, and its gradient, against
whole-number buckets and 64-bit sums.  The bias is the table's value rounded once: equal bit for
bit.  A gradient's sum has at most 128 f32 additions behind one another (64 rows a thread, 8
phases, 33 + 6 over a window, then double), so it is off by at most 128 * 2^-24 of the terms'
magnitudes, and half a step of the result."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError
from operator_refs import bucket, buckets_of, off

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]
FIRST = 4   # rows in front of the bias's


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _server(heads, buckets, seed=0, stride=1):
    s = psa.Server(0, 1)
    s.CreateTable(5, psa.TableInfo(row_capacity=heads, max_rows=FIRST + buckets + 3, row_stride=stride, row_offset=1))
    w = np.random.RandomState(seed).normal(size=(FIRST + buckets + 3, heads)).astype(np.float32)
    s.load_rows(5, 1, w)
    return s, torch.from_numpy(w[FIRST:FIRST + buckets]), 1 + FIRST * stride


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("buckets,distance", [(32, 128), (8, 100), (64, 513), (4, 3), (256, 5000)])
def test_every_distance_has_its_bucket(buckets, distance, both):
    """One head whose row j holds j: distances past the last border both ways, borders included."""
    s, _, row = _server(1, buckets)
    s.load_rows(5, row, np.arange(buckets, dtype=np.float32)[:, None])
    n = distance + 40
    got = s.position_bias(5, row, buckets, distance, both).forward(1, 2 * n + 1, n)[0, 0].cpu().numpy()
    want = [bucket(r, buckets, distance, both) for r in range(-n, n + 1)]
    assert got.astype(int).tolist() == want
    s.close()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("q,k,begin", [(1, 1, 0), (1, 8191, 8190), (3, 2049, 0), (17, 33, 16), (77, 131, 54), (130, 9, -5),
                                       (40, 264, 1 << 33)])
def test_forward(dt, q, k, begin):
    s, w, row = _server(5, 32, seed=q)
    bias = s.position_bias(5, row, 32, 128, True)
    got = bias.forward(q, k, begin, dt)
    at = buckets_of(q, k, begin, 32, 128, True) if abs(begin) < 1 << 20 else torch.full((q, k), 15)
    want = w.t()[:, at].to(dt)
    assert got.dtype == dt and torch.equal(got.cpu(), want)
    s.close()


@pytest.mark.parametrize("dt", DT)
def test_forward_into_strides(dt):
    """Padded rows, rows at odd addresses, and heads inside queries; what lies between stays."""
    q, k, H = 19, 45, 3
    s, w, row = _server(H, 16, stride=2)
    bias = s.position_bias(5, row, 16, 64, False)
    want = w.t()[:, buckets_of(q, k, 3, 16, 64, False)].to(dt)
    buf = torch.full((H, q + 2, k + 6), 9.0, dtype=dt, device="cuda")
    bias.forward(q, k, 3, out=buf[:, 1:q + 1, 3:k + 3])
    full = torch.full(buf.shape, 9.0, dtype=dt)
    full[:, 1:q + 1, 3:k + 3] = want
    assert torch.equal(buf.cpu(), full)
    inner = torch.zeros(q, H, k, dtype=dt, device="cuda")
    bias.forward(q, k, 3, out=inner.transpose(0, 1))
    assert torch.equal(inner.transpose(0, 1).cpu(), want)
    s.close()


def _check_grad(got, d, at, buckets, gain):
    d = d.double().cpu()
    hot = torch.nn.functional.one_hot(at.flatten(), buckets).double()
    B, H = d.shape[:2]
    want = gain * (d.sum(0).reshape(H, -1) @ hot).t()
    mag = abs(gain) * (d.abs().sum(0).reshape(H, -1) @ hot).t()
    assert off(got, want, 128 * 2.0 ** -24 * mag + 2.0 ** -24 * want.abs() + 1e-40) <= 1


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,H,q,k,begin,both", [(1, 1, 1, 1, 0, True), (2, 12, 77, 131, 54, False), (1, 3, 1, 4099, 4098, True),
                                                (3, 2, 300, 41, 0, True), (1, 2, 257, 2050, -3, False),
                                                (2, 1, 513, 1024, 511, True)])
def test_gradient(dt, B, H, q, k, begin, both):
    s, _, row = _server(H, 32)
    d = torch.randn(B, H, q, k, generator=torch.Generator().manual_seed(q * k)).to(dt).cuda()
    got = s.position_bias(5, row, 32, 128, both).backward(d, begin, -0.25)
    _check_grad(got, d, buckets_of(q, k, begin, 32, 128, both), 32, -0.25)
    again = s.position_bias(5, row, 32, 128, both).backward(d, begin, -0.25)
    assert torch.equal(got, again)   # a fixed order
    s.close()


@pytest.mark.parametrize("dt", DT)
def test_gradient_of_strided_and_broadcast_scores(dt):
    q, k, H = 30, 50, 4
    s, _, row = _server(H, 8)
    bias = s.position_bias(5, row, 8, 20, True)
    at = buckets_of(q, k, 0, 8, 20, True)
    buf = torch.randn(2, q, H, k + 5, device="cuda").to(dt)
    d = buf.permute(0, 2, 1, 3)[..., 2:k + 2]
    _check_grad(bias.backward(d), d, at, 8, 1.0)
    shared = buf[:1, :, :1, :k].permute(0, 2, 1, 3).expand(3, H, q, k)   # one plane for every batch and head
    _check_grad(bias.backward(shared), shared, at, 8, 1.0)
    s.close()


def test_gradient_against_differences():
    """The loss sum(c * bias^2) / 2 has d = c * bias; moving one bucket's value changes it so."""
    q, k, H, buckets = 9, 23, 2, 8
    s, w, row = _server(H, buckets)
    bias = s.position_bias(5, row, buckets, 16, True)
    c = torch.randn(H, q, k, generator=torch.Generator().manual_seed(1)).cuda()

    def loss():
        return float((c.double() * bias.forward(q, k, 0).double() ** 2).sum() / 2)

    grad = bias.backward(c * bias.forward(q, k, 0)).cpu()
    for j, h in [(0, 0), (3, 1), (5, 0), (7, 1)]:
        side = []
        for step in (0.25, -0.25):   # the loss is a parabola: central differences are exact but for rounding
            moved = w[j:j + 1].clone()
            moved[0, h] += step
            s.load_rows(5, row + j, moved.numpy())
            side.append(loss())
        s.load_rows(5, row + j, w[j:j + 1].numpy())
        slope = (side[0] - side[1]) / 0.5
        assert abs(slope - float(grad[j, h])) <= 1e-3 * (1 + abs(slope))
    s.close()


def test_masked_places_and_empty_shapes():
    """An Inf or a NaN reaches its own bucket and head only; lengths of zero give zero rows."""
    s, _, row = _server(2, 8)
    bias = s.position_bias(5, row, 8, 16, True)
    at = buckets_of(6, 7, 0, 8, 16, True)
    d = torch.zeros(1, 2, 6, 7, device="cuda")
    d[0, 1, 2, 2] = float("nan")   # bucket 0
    d[0, 0, 0, 6] = float("inf")
    got = bias.backward(d).cpu()
    assert torch.isnan(got[0, 1]) and got[int(at[0, 6]), 0] == float("inf")
    got[0, 1] = got[int(at[0, 6]), 0] = 0
    assert torch.equal(got, torch.zeros(8, 2))
    for shape in [(0, 2, 3, 4), (1, 2, 0, 4), (1, 2, 3, 0)]:
        assert torch.equal(bias.backward(torch.zeros(shape, device="cuda")).cpu(), torch.zeros(8, 2))
    assert bias.forward(0, 5).shape == (2, 0, 5) and bias.forward(5, 0).shape == (2, 5, 0)
    s.sync()
    s.close()


@pytest.mark.parametrize("shape", [(0, 2, 3, 4), (1, 2, 0, 4), (1, 2, 3, 0), (2, 2, 300, 0)])
def test_empty_scores_leave_the_scratch_unread(shape):
    s, _, row = _server(2, 8)
    work = torch.full((1 << 16,), float("nan"), device="cuda")
    got = s.position_bias(5, row, 8, 16, True).backward(torch.zeros(shape, device="cuda"), work=work)
    assert torch.equal(got.cpu(), torch.zeros(8, 2))
    s.close()


def test_refusals():
    s, _, row = _server(3, 8)
    for args in [(5, row, 7, 16, True), (5, row, 1, 16, False), (5, row, 8, 2, True), (5, row, 258, 512, True),
                 (5, row, 8, (1 << 20) + 1, True)]:
        with pytest.raises(PsxError) as e:
            s.position_bias(*args)
        assert e.value.status == 1
    for args, status in [((6, row, 8, 16, True), 3), ((5, 0, 8, 16, True), 5), ((5, row + 4, 8, 16, True), 5)]:
        with pytest.raises(PsxError) as e:
            s.position_bias(*args)
        assert e.value.status == status
    s.CreateTable(7, psa.TableInfo(row_capacity=3, max_rows=16, dtype=psa.F64))
    with pytest.raises(PsxError) as e:
        s.position_bias(7, 0, 8, 16, True)
    assert e.value.status == 10
    bias = s.position_bias(5, row, 8, 16, True)
    out = torch.zeros(3, 4, 8, device="cuda")
    for bad in [out[:2], out.double(), out.cpu(), out.transpose(1, 2), out[:, :, ::2], out[:1].expand(3, 4, 8)]:
        with pytest.raises(PsxError) as e:
            bias.forward(4, bad.shape[2] if bad.shape[2] != 4 else 8, out=bad)
        assert e.value.status == 1
    with pytest.raises(PsxError):
        bias.forward(4, 8, 1 << 41, out=out)
    with pytest.raises(PsxError):
        bias.backward(torch.zeros(1, 2, 4, 8, device="cuda"))
    with pytest.raises(PsxError) as e:   # one row as 3 * 2^48 scores
        bias.backward(torch.zeros(1 << 24, device="cuda").expand(3, 1 << 24, 1 << 24))
    assert e.value.status == 10
    bias.close()
    with pytest.raises(PsxError):
        bias.forward(4, 8)
    late = s.position_bias(5, row, 8, 16, True)
    s.close()
    with pytest.raises(PsxError):
        late.forward(4, 8)
    late.close()
