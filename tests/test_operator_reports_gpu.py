"""What only the GPU sees of a batch of requests comes out of the next psx_sync, and of nothing
else: not lost behind an apply's error, not out of a row read, a load or the next operator."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError, wire
from operator_refs import Batch, off

pytestmark = pytest.mark.gpu
A, B = 11, 12
UNKNOWN_TABLE, MALFORMED = 3, 4


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture
def case():
    b = Batch(31, [10], [0], [4, 4], 40, 48, torch.float32)
    s = psa.Server(0, 1, [1])
    for t, w in ((A, b.a), (B, b.b)):
        s.CreateTable(t, psa.TableInfo(row_capacity=w.shape[1], max_rows=b.rows))
        s.load_rows(t, 0, w.numpy())
    yield b, s, s.create_adapters(A, B, b.adapters())
    s.close()


def _ids(cuts, which):
    return torch.tensor(cuts, dtype=torch.int32).cuda(), torch.tensor(which, dtype=torch.int32).cuda()


def _status(call):
    try:
        call()
    except PsxError as e:
        return e.status
    return 0


def _rejected(s, version):
    """An apply call that the GPU rejects."""
    bad = torch.from_numpy(np.array(wire.dense_stream_np(99, np.arange(3, dtype=np.int32), np.ones((3, 40), np.float32)),
                                    copy=True)).cuda()
    torch.cuda.synchronize()
    s.apply_device([(bad.data_ptr(), bad.numel(), 1, version)])
    return bad


@pytest.mark.parametrize("cuts,which", [([0, 3, 2, 10], [0, 0, 0]), ([0, 3, 5, 10], [0, 2, 0])])
def test_an_apply_error_does_not_hide_the_report(case, cuts, which):
    b, s, ads = case
    x = b.x.cuda()
    ads.forward(x, *_ids(cuts, which))
    bad = _rejected(s, 0)
    assert [_status(s.sync) for _ in range(3)] == [UNKNOWN_TABLE, MALFORMED, 0]
    del bad


def test_no_other_call_takes_the_report(case):
    b, s, ads = case
    x = b.x.cuda()
    good = _ids([0, 10], [0])
    ads.forward(x, *_ids([0, 3, 5, 11], [0, 0, 0]))
    assert np.array_equal(s.read_rows(A, 0, b.rows), b.a.numpy())
    s.load_rows(A, 0, (2 * b.a).numpy())   # is loaded
    b.a = 2 * b.a
    assert np.array_equal(s.read_rows(A, 0, b.rows), b.a.numpy())
    got = ads.forward(x, *good, base=b.base.cuda())[0]
    want, tol = b.forward(torch.zeros(10, 48))
    assert off(got, want, tol) <= 1
    assert [_status(s.sync) for _ in range(2)] == [MALFORMED, 0]


def test_the_report_of_a_call_before_another_calls_rejection(case):
    """The rejection settles inside an operator, which returns it; the report stays."""
    b, s, ads = case
    x = b.x.cuda()
    ads.forward(x, *_ids([0, 3, 5, 10], [0, -2, 0]))
    bad = _rejected(s, 0)
    assert _status(lambda: ads.forward(x, *_ids([0, 10], [0]))) == UNKNOWN_TABLE
    assert [_status(s.sync) for _ in range(2)] == [MALFORMED, 0]
    del bad


def test_replays_are_reported_each_time(case):
    b, s, ads = case
    x, out = b.x.cuda(), torch.zeros(10, 48, device="cuda")
    begin, which = _ids([0, 10], [0])
    shrunk = ads.forward(x, begin, which, out=out)[1]
    s.sync()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ads.forward(x, begin, which, out=out, shrunk=shrunk)
    for adapter, want in ((0, 0), (7, MALFORMED), (0, 0), (0, 0), (-3, MALFORMED), (1, 0)):
        which.fill_(adapter)
        g.replay()
        torch.cuda.synchronize()
        assert _status(s.sync) == want


def test_a_request_with_a_bad_adapter_is_taken_as_one_without(case):
    b, s, ads = case
    x, dy, base = b.x.cuda(), b.dy.cuda(), b.base.cuda()
    cuts = [0, 3, 5, 10]
    got = []
    for which in ([0, 2, 1], [0, -1, 1]):
        ids = _ids(cuts, which)
        out, shrunk = ads.forward(x, *ids, base=base)
        dx = torch.zeros_like(x)
        got.append((out, dx) + ads.backward(x, dy, shrunk, *ids, out=dx))
        assert _status(s.sync) == (MALFORMED if 2 in which else 0)
    assert all(torch.equal(p, q) for p, q in zip(*got))
    assert torch.equal(got[0][0][3:5], base[3:5])


def test_calls_without_tokens_or_requests_look_at_no_offsets(case):
    b, s, ads = case
    none = torch.zeros(0, 40, device="cuda")
    out, shrunk = ads.forward(none, *_ids([0, 5], [9]))
    ga, gb = ads.backward(none, torch.zeros(0, 48, device="cuda"), shrunk, *_ids([0, 5], [9]))
    assert not ga.any() and not gb.any()
    ads.forward(b.x.cuda(), *_ids([77], []))
    assert _status(s.sync) == 0
