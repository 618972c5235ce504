"""Low-rank adapters of many requests (rows of two tables), forward and backward, against
64-bit products.  Tolerances count the f32 additions of each sum (operator_refs.F23 each), the
parts left out of expand's factors for 16-bit outputs, and the output's rounding."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError, _abi
from operator_refs import Batch, checkpoint, off
from oracle.oracle import OracleServer, DENSE, F32

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]
A, B = 11, 12


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib, oracle_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _server(b, stride=1, offset=0):
    s = psa.Server(0, 1, [1])
    for t, w in ((A, b.a), (B, b.b)):
        s.CreateTable(t, psa.TableInfo(row_capacity=w.shape[1], max_rows=b.rows, row_stride=stride, row_offset=offset))
        s.load_rows(t, offset, w.numpy())
    return s


def _ids(b):
    return (torch.tensor(b.begin, dtype=torch.int32).cuda(), torch.tensor(b.which, dtype=torch.int32).cuda())


def _adapters(s, b, stride=1, offset=0):
    return s.create_adapters(A, B, [(offset + stride * f, r, sc) for f, r, sc in b.adapters()])


def _run(b, base=True, ck=False, gain=-0.5, stride=1, offset=0):
    """Forward and backward, all outputs against the reference."""
    s = _server(b, stride, offset)
    ads = _adapters(s, b, stride, offset)
    begin, which = _ids(b)
    x, dy = b.x.cuda(), b.dy.cuda()
    out = torch.full((b.T, b.d_out), 7.0, dtype=b.dtype, device="cuda")
    got, shrunk = ads.forward(x, begin, which, base=b.base.cuda() if base else None, out=out)
    assert got is out
    want, tol = b.forward(torch.full((b.T, b.d_out), 7.0), base)
    assert off(out, want, tol) <= 1
    kept = s.checkpoint_store(x) if ck else x
    dx = torch.full((b.T, b.d_in), 7.0, dtype=b.dtype, device="cuda")
    ga, gb = ads.backward(kept, dy, shrunk, begin, which, base=b.dbase.cuda() if base else None, out=dx, scale=gain)
    want, tol = b.backward(torch.full((b.T, b.d_in), 7.0), gain, checkpoint(b.x) if ck else None, base)
    for name, g in (("dx", dx), ("grad_a", ga), ("grad_b", gb)):
        assert off(g, want[name], tol[name]) <= 1, name
    again = ads.backward(kept, dy, shrunk, begin, which, scale=gain)
    assert torch.equal(again[0], ga) and torch.equal(again[1], gb)   # without dx, and in the same order
    s.sync()
    s.close()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lengths,which,ranks,d_in,d_out", [
    ([1], [0], [1], 1, 1),                                        # the smallest
    ([1] * 9, [0, 1, 2, 0, -1, 1, 2, 2, 0], [16, 4, 7], 256, 320),   # a decode step, shared adapters, one without
    ([5, 0, 19, 1, 0, 33, 16], [1, 0, 1, 0, 1, -1, 0], [5, 12], 129, 65),   # empty requests, odd widths
    ([0, 0, 0], [0, 1, 0], [3, 4], 16, 24),                       # nothing at all
    ([40], [-1], [8], 33, 70),                                    # no adapter
    ([70, 3], [1, 0], [33, 64], 95, 130),                         # ranks that fill no tile
    ([17, 40, 8], [2, 0, 2], [65, 16, 150], 192, 67),             # ranks past one group
])
def test_small(dt, lengths, which, ranks, d_in, d_out):
    _run(Batch(1, lengths, which, ranks, d_in, d_out, dt, lead=2, tail=3))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("base,ck", [(False, False), (True, True), (False, True)])
def test_base_and_checkpoint(dt, base, ck):
    _run(Batch(2, [30, 2, 61], [1, 0, 1], [6, 20], 200, 101, dt, tail=1), base=base, ck=ck)


@pytest.mark.parametrize("dt", DT)
def test_many_requests(dt):
    """More requests than lanes of a wave, and than a square of them."""
    r = np.random.RandomState(3)
    n = 300
    lengths = r.choice([0, 1, 1, 2, 5], size=n).tolist()
    _run(Batch(4, lengths, r.randint(-1, 70, size=n).tolist(), r.randint(1, 18, size=70).tolist(), 72, 40, dt))


def test_very_many_requests():
    r = np.random.RandomState(5)
    n = 5000
    _run(Batch(6, r.choice([0, 0, 1], size=n).tolist(), r.randint(-1, 3, size=n).tolist(), [2, 3, 4], 24, 40, torch.bfloat16,
               tail=1))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("ck", [False, True])
def test_long(dt, ck):
    """Past 1024 tokens: wide tiles, gradients in several parts, an adapter whose requests lie apart."""
    _run(Batch(7, [1100, 37, 900, 1, 600], [0, 1, 0, 2, 1], [16, 40, 3], 136, 200, dt, tail=4), ck=ck)


@pytest.mark.parametrize("ranks", [[16], [32], [64], [128]])
def test_ranks_of_whole_tiles(ranks):
    _run(Batch(8, [200], [0], ranks, 512, 768, torch.bfloat16))


def test_rows_that_step():
    """A shard of every third row id, from 5 on."""
    _run(Batch(9, [8, 9], [1, 0], [4, 6], 32, 48, torch.float32), stride=3, offset=5)


@pytest.mark.parametrize("dt", DT)
def test_strides(dt):
    """Rows apart from one another and at odd addresses; what lies between stays."""
    b = Batch(10, [21, 18], [0, 1], [5, 9], 70, 90, dt, x_pad=3)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)

    def apart(t):
        buf = torch.full((t.shape[0] + 2, t.shape[1] + 7), 7.0, dtype=dt, device="cuda")
        buf[1:-1, 3:-4] = t.cuda()
        return buf, buf[1:-1, 3:-4]

    obuf, out = apart(torch.full((b.T, 90), 7.0))
    _, shrunk = ads.forward(apart(b.x)[1], begin, which, base=apart(b.base)[1], out=out)
    want, tol = b.forward(torch.zeros(b.T, 90))
    assert off(out, want, tol) <= 1
    ibuf, io = apart(b.base)
    ads.forward(apart(b.x)[1], begin, which, base=io, out=io)   # in place
    assert torch.equal(io, out)
    dbuf, dx = apart(b.dbase)
    ga, gb = ads.backward(apart(b.x)[1], apart(b.dy)[1], shrunk, begin, which, base=dx, out=dx)
    want, tol = b.backward(torch.zeros(b.T, 70), 1.0)
    for name, g in (("dx", dx), ("grad_a", ga), ("grad_b", gb)):
        assert off(g, want[name], tol[name]) <= 1, name
    for buf in (obuf, ibuf, dbuf):
        edge = buf.clone()
        edge[1:-1, 3:-4] = 7.0
        assert bool((edge == 7.0).all())
    s.close()


def test_values_that_are_not_finite_stay_in_their_request():
    """A row behind the last request and a request without an adapter hold NaN and Inf: nobody
    else sees them; a token that does turns its own row alone."""
    b = Batch(11, [20, 9, 30], [0, -1, 0], [5], 64, 64, torch.bfloat16, tail=2)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    x, dy = b.x.clone(), b.dy.clone()
    for t in (x, dy):
        t[20:29] = float("inf")
        t[59:] = float("nan")
    out, shrunk = ads.forward(x.cuda(), begin, which, out=torch.zeros(b.T, 64, dtype=b.dtype, device="cuda"))
    dx = torch.zeros(b.T, 64, dtype=b.dtype, device="cuda")
    got = (dx,) + ads.backward(x.cuda(), dy.cuda(), shrunk, begin, which, out=dx)
    clean = ads.forward(b.x.cuda(), begin, which)
    dx2 = torch.zeros_like(dx)
    want = (dx2,) + ads.backward(b.x.cuda(), b.dy.cuda(), clean[1], begin, which, out=dx2)
    assert torch.equal(out, clean[0]) and all(torch.equal(g, w) for g, w in zip(got, want))
    x[3, 10] = float("inf")
    hit = ads.forward(x.cuda(), begin, which)[0].cpu()
    rows = [t for t in range(b.T) if t != 3]
    assert not torch.isfinite(hit[3]).any() and torch.equal(hit[rows][:59], clean[0].cpu()[rows][:59])
    s.close()


def test_gradients_against_differences():
    """The loss sum(c * out): moving one row value (or one input) moves it by the gradient times
    the step, exactly but for rounding, since out is linear in each."""
    b = Batch(12, [6, 4], [0, 1], [2, 3], 24, 20, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    c = b.dy.cuda()

    def loss(x):
        return float((ads.forward(x, begin, which)[0].double() * c.double()).sum())

    x = b.x.cuda()
    out, shrunk = ads.forward(x, begin, which)
    dx = torch.zeros_like(x)
    ga, gb = ads.backward(x, c, shrunk, begin, which, out=dx)
    for table, w, grad in ((A, b.a, ga), (B, b.b, gb)):
        for k, col in [(0, 0), (1, 7), (3, 19), (4, 3)]:
            row = int(ads.row_ids[k])
            side = []
            for step in (0.5, -0.5):
                moved = w[row:row + 1].clone()
                moved[0, col] += step
                s.load_rows(table, row, moved.numpy())
                side.append(loss(x))
            s.load_rows(table, row, w[row:row + 1].numpy())
            assert abs(side[0] - side[1] - float(grad[k, col])) <= 1e-4
    for t, col in [(0, 0), (7, 23), (9, 5)]:
        side = []
        for step in (0.5, -0.5):
            moved = x.clone()
            moved[t, col] += step
            side.append(loss(moved))
        assert abs(side[0] - side[1] - float(dx[t, col])) <= 1e-4
    s.close()


def test_a_training_step_through_the_server():
    """Forward, backward, the increments packed and applied, the next forward from the new rows:
    the tables follow the oracle bit for bit."""
    b = Batch(13, [50, 30, 20], [0, 1, 0], [4, 8], 96, 64, torch.bfloat16)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    orc = OracleServer([1])
    for t, w in ((A, b.a), (B, b.b)):
        orc.create_table(t, DENSE, F32, w.shape[1])
        orc.load_dense_rows(t, 0, w.numpy())
    for version in range(3):
        out, shrunk = ads.forward(b.x.cuda(), begin, which, base=b.base.cuda())
        want, tol = b.forward(torch.zeros(b.T, b.d_out))
        assert off(out, want, tol) <= 1
        ga, gb = ads.backward(s.checkpoint_store(b.x.cuda()), b.dy.cuda(), shrunk, begin, which, scale=-0.125)
        msg = s.pack_stream([dict(table_id=t, dtype=psa.F32, dense_serialized=True, row_ids=ads.row_ids, oplogs=g)
                             for t, g in ((A, ga), (B, gb))])
        s.apply_device([(msg.data_ptr(), msg.numel(), 1, version)])   # the next forward settles it
        assert orc.apply_stream(msg.cpu().numpy(), 1, version) == 0
        # the rows that the next forward reads, and this test's reference of it
        fresh, _ = ads.forward(b.x.cuda(), begin, which, base=b.base.cuda())
        b.a = torch.from_numpy(orc.read_dense_rows(A, 0, b.rows).copy())
        b.b = torch.from_numpy(orc.read_dense_rows(B, 0, b.rows).copy())
        want, tol = b.forward(torch.zeros(b.T, b.d_out))
        assert off(fresh, want, tol) <= 1
    for t, w in ((A, b.a), (B, b.b)):
        assert np.array_equal(s.read_rows(t, 0, b.rows).view(np.uint32), w.numpy().view(np.uint32))
    s.close()


def test_writers_wait_for_readers():
    """A long forward pass on a side stream, then rows loaded and an apply: the pass saw the rows
    that were there when it was launched."""
    b = Batch(14, [4000], [0], [64], 1024, 1024, torch.bfloat16)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    x, base = b.x.cuda(), b.base.cuda()
    want = ads.forward(x, begin, which, base=base)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    zero = np.zeros((b.rows, 1024), np.float32)
    ids = torch.arange(b.rows, dtype=torch.int32, device="cuda")
    big = torch.full((b.rows, 1024), 1e3, device="cuda")
    msg = s.pack_stream([dict(table_id=t, dtype=psa.F32, dense_serialized=True, row_ids=ids, oplogs=big) for t in (A, B)])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [ads.forward(x, begin, which, base=base)[0] for _ in range(4)]
    s.apply_device([(msg.data_ptr(), msg.numel(), 1, 0)])
    with torch.cuda.stream(side):
        changed = ads.forward(x, begin, which, base=base)[0]
    s.load_rows(A, 0, zero)
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs) and not torch.equal(changed, want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        none = ads.forward(x, begin, which, base=base)[0]
    side.synchronize()
    assert torch.equal(none, base)
    s.close()


def test_graph_replays():
    """Forward and backward in one graph: replays with other inputs, other requests and other rows,
    eager work between them, each against the eager calls; two graphs with their own buffers."""
    b = Batch(15, [3, 40, 1, 25], [1, 0, -1, 1], [8, 20], 160, 96, torch.bfloat16)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    x, dy, base = b.x.cuda(), b.dy.cuda(), b.base.cuda()
    s.sync()

    def step():
        out, shrunk = ads.forward(x, begin, which, base=base)
        dx = torch.zeros_like(x)
        return (out, dx) + ads.backward(s.checkpoint_store(x), dy, shrunk, begin, which, out=dx)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    r = np.random.RandomState(1)
    for k in range(4):
        x.copy_(torch.from_numpy(r.normal(size=x.shape)).bfloat16())
        cuts = np.sort(r.randint(0, b.T + 1, size=5)).astype(np.int32)
        begin.copy_(torch.from_numpy(cuts))
        which.copy_(torch.from_numpy(r.randint(-1, 2, size=4).astype(np.int32)))
        if k == 2:
            s.load_rows(A, 0, (2 * b.a).numpy())
        for g, _ in graphs:
            g.replay()
        eager = step()
        torch.cuda.synchronize()
        for _, got in graphs:
            inside = slice(int(cuts[0]), int(cuts[-1]))
            assert torch.equal(got[0][inside], eager[0][inside]) and all(torch.equal(p, q) for p, q in zip(got[1:], eager[1:]))
    s.sync()
    s.close()


def test_a_capture_refuses_calls_in_flight():
    b = Batch(16, [4], [0], [2], 8, 8, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    x, out = b.x.cuda(), torch.zeros(4, 8, device="cuda")
    shrunk = ads.forward(x, begin, which, out=out)[1]
    msg = s.pack_stream([dict(table_id=A, dtype=psa.F32, dense_serialized=True, row_ids=ads.row_ids,
                              oplogs=torch.ones(2, 8, device="cuda"))])
    s.apply_device([(msg.data_ptr(), msg.numel(), 1, 0)])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(PsxError) as e:
            ads.forward(x, begin, which, out=out, shrunk=shrunk)
        out.zero_()
    assert e.value.status == 10
    s.sync()
    s.close()


@pytest.mark.parametrize("cuts,which", [([0, 3, 2, 10], [0, 0, 0]), ([0, 3, 5, 11], [0, 0, 0]), ([-1, 3, 5, 10], [0, 0, 0]),
                                        ([0, 3, 5, 10], [0, 2, 0]), ([0, 3, 5, 10], [0, -2, 0])])
def test_bad_requests_are_reported_by_sync(cuts, which):
    b = Batch(17, [10], [0], [4, 4], 40, 48, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    begin, w = torch.tensor(cuts, dtype=torch.int32).cuda(), torch.tensor(which, dtype=torch.int32).cuda()
    out, shrunk = ads.forward(b.x.cuda(), begin, w)
    with pytest.raises(PsxError) as e:
        s.sync()
    assert e.value.status == 4
    s.sync()   # once
    dx = torch.zeros(10, 40, device="cuda")
    ads.backward(b.x.cuda(), b.dy.cuda(), shrunk, begin, w, out=dx)
    with pytest.raises(PsxError) as e:
        s.sync()
    assert e.value.status == 4
    good = torch.tensor([0, 10], dtype=torch.int32).cuda(), torch.tensor([0], dtype=torch.int32).cuda()
    got = ads.forward(b.x.cuda(), *good, base=b.base.cuda())[0]
    want, tol = b.forward(torch.zeros(10, 48))
    assert off(got, want, tol) <= 1
    s.sync()
    s.close()


def test_sets_that_are_refused():
    b = Batch(18, [4], [0], [4, 4], 8, 8, torch.float32)
    s = _server(b)
    s.CreateTable(20, psa.TableInfo(row_capacity=8, max_rows=b.rows, dtype=psa.F64))
    s.CreateTable(21, psa.TableInfo(row_kind=psa.ROW_SORTED_MAP, dtype=psa.I32, oplog_dense_serialized=False, max_rows=8,
                                    max_entries=8))
    s.CreateTable(22, psa.TableInfo(row_capacity=8, max_rows=b.rows, row_stride=2))
    for args, status in [((A, B, []), 1), ((A, B, [(0, 0, 1.0)]), 1), ((A, B, [(0, 257, 1.0)]), 1),
                         ((A, B, [(0, 2, float("nan"))]), 1), ((A, B, [(0, 3, 1.0), (2, 2, 1.0)]), 1),
                         ((A, B, [(b.rows - 1, 2, 1.0)]), 5), ((A, B, [(-1, 2, 1.0)]), 5), ((A, 99, [(0, 2, 1.0)]), 3),
                         ((A, 20, [(0, 2, 1.0)]), 10), ((21, B, [(0, 2, 1.0)]), 10), ((A, 22, [(0, 2, 1.0)]), 1),
                         ((A, B, [(0, 1, 1.0)] * 4097), 1)]:
        with pytest.raises(PsxError) as e:
            s.create_adapters(*args)
        assert e.value.status == status, args[2][:3]
    ads = _adapters(s, b)
    n, p = ctypes.c_int32(), ctypes.c_void_p()
    assert s._L.psx_adapters_info(ads._h, ctypes.byref(n), ctypes.byref(p)) == 0
    assert n.value == 8 and p.value and ads.row_ids.tolist() == [3, 4, 5, 6, 8, 9, 10, 11]
    ads.close()
    with pytest.raises(PsxError):
        ads.forward(b.x.cuda(), *_ids(b))
    late = _adapters(s, b)
    s.close()
    with pytest.raises(PsxError):
        late.forward(b.x.cuda(), *_ids(b))


def test_calls_that_are_refused():
    b = Batch(19, [6], [0], [4], 16, 24, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    x, dy, base = b.x.cuda(), b.dy.cuda(), b.base.cuda()
    out, shrunk = ads.forward(x, begin, which, base=base)
    both = torch.zeros(6, 64, device="cuda")
    for kw in [dict(x=b.x), dict(x=x.double()), dict(x=x.half()), dict(x=x[:, :8]), dict(x=x.t()), dict(base=base[:5]),
               dict(out=out[:5]), dict(out=base.half()), dict(out=out[:1].expand(6, 24)), dict(begin=begin.long()),
               dict(begin=begin[:1]), dict(which=which.cpu()), dict(shrunk=shrunk[:3]), dict(shrunk=shrunk[1:]),
               dict(x=both[:, :16], out=both[:, 8:32]), dict(base=both[:, :24], out=both[:, 1:25])]:
        a = dict(x=x, begin=begin, which=which, base=base, out=out, shrunk=shrunk)
        a.update(kw)
        with pytest.raises(PsxError) as e:
            ads.forward(a["x"], a["begin"], a["which"], base=a["base"], out=a["out"], shrunk=a["shrunk"])
        assert e.value.status == 1, kw.keys()
    dx = torch.zeros(6, 16, device="cuda")
    ck = s.checkpoint_store(x[:5])
    for kw in [dict(dy=dy.half()), dict(dy=dy[:, :16]), dict(x=ck), dict(out=dy[:, :16]), dict(out=x), dict(out=dx.half()),
               dict(out=None, base=dx), dict(grad_a=torch.zeros(4, 15, device="cuda")), dict(work=shrunk[:1]),
               dict(grad_b=torch.zeros(4, 24, device="cuda").half())]:
        a = dict(x=x, dy=dy, out=dx, base=None, grad_a=None, grad_b=None, work=None)
        a.update(kw)
        with pytest.raises(PsxError) as e:
            ads.backward(a["x"], a["dy"], shrunk, begin, which, base=a["base"], out=a["out"], grad_a=a["grad_a"],
                         grad_b=a["grad_b"], work=a["work"])
        assert e.value.status == 1, kw.keys()
    # the C call itself: both activations, or none
    L, P = s._L, ctypes.byref
    m = lambda t: _abi.psx_matrix(t.data_ptr(), 0, 0, t.shape[0], t.shape[1], t.stride(0))  # noqa: E731
    r = _abi.psx_requests(begin.data_ptr(), which.data_ptr(), 1, 0)
    whole = s.checkpoint_store(x)
    ga, gb, work = torch.zeros(4, 16, device="cuda"), torch.zeros(4, 24, device="cuda"), torch.zeros(1 << 16, device="cuda")
    for xm, c in [(m(x), whole.buffer.data_ptr()), (None, None)]:
        assert L.psx_adapters_backward(ads._h, P(r), P(xm) if xm else None, c, P(m(dy)), shrunk.data_ptr(), None, None,
                                       ga.data_ptr(), gb.data_ptr(), 1.0, work.data_ptr(), None) == 1
    far = _abi.psx_matrix(x.data_ptr(), 0, 0, 6, 16, (16 << 20) + 1)   # rows more than 64 MiB apart
    apart = _abi.psx_matrix(base.data_ptr(), 0, 0, 6, 24, (16 << 20) + 1)
    for xm, bm in [(far, None), (m(x), P(apart))]:
        assert L.psx_adapters_forward(ads._h, P(r), P(xm), bm, P(m(out)), shrunk.data_ptr(), None) == 1
        assert b"64 MiB" in L.psx_last_error(s._ctx)
    many = _abi.psx_requests(begin.data_ptr(), which.data_ptr(), 1 << 24, 0)   # 2^24 blocks of 256 threads
    assert L.psx_adapters_forward(ads._h, P(many), P(m(x)), None, P(m(out)), shrunk.data_ptr(), None) == 10
    size = ctypes.c_size_t()
    assert L.psx_adapters_sizes(ads._h, 1 << 30, P(size), None) == 10 and L.psx_adapters_sizes(ads._h, -1, P(size), None) == 1
    bad = _abi.psx_requests(begin.data_ptr() + 2, which.data_ptr(), 1, 0)
    assert L.psx_adapters_forward(ads._h, P(bad), P(m(x)), None, P(m(out)), shrunk.data_ptr(), None) == 1
    s.sync()
    s.close()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("lengths,which,ranks,d_in,d_out,ck", [
    ([20, 3, 1, 16], [1, 0, 0, -1], [5, 40], 4100, 2050, False),        # few tokens: x's width in parts
    ([7000, 1500, 0, 700], [1, 0, 1, 2], [16, 70, 3], 1030, 520, False),   # a long batch: parts joined, the widest tiles
    ([7000, 1500, 0, 700], [1, 0, 1, 0], [16, 30], 1030, 520, True),
    ([8200], [0], [9], 600, 72, False),
])
def test_parts_of_a_width(dt, lengths, which, ranks, d_in, d_out, ck):
    _run(Batch(21, lengths, which, ranks, d_in, d_out, dt, tail=2), ck=ck)


@pytest.mark.parametrize("ranks", [[3], [20, 5], [40, 256]])
@pytest.mark.parametrize("width", [64, 1024, 4100])
def test_buffers_serve_fewer_tokens(ranks, width):
    b = Batch(23, [1], [0], ranks, width, 96, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    last = (0, 0)
    counts = sorted({max(0, 2 ** k + j) for k in range(18) for j in (-1, 0, 1, 33)} | set(range(5900, 6500, 7)))
    for t in counts:
        now = ads.sizes(t)
        assert now[0] >= last[0] and now[1] >= last[1], t
        last = now
    s.close()


def test_two_calls_at_once():
    """The same set on two streams with buffers of their own, outputs in the place of their bases."""
    b = Batch(22, [300, 200], [0, 1], [24, 8], 640, 512, torch.bfloat16)
    s = _server(b)
    ads = _adapters(s, b)
    begin, which = _ids(b)
    other = which.flip(0).contiguous()
    x, dy = b.x.cuda(), b.dy.cuda()

    def step(ids, out, dx):
        shrunk = ads.forward(x, begin, ids, base=out, out=out)[1]
        return (out, dx) + ads.backward(x, dy, shrunk, begin, ids, base=dx, out=dx)

    want = [step(ids, b.base.cuda(), b.dbase.cuda()) for ids in (which, other)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rounds = [[(b.base.cuda(), b.dbase.cuda()) for _ in range(3)] for _ in streams]
    got = []
    torch.cuda.synchronize()
    for k in range(3):
        for i, ids in enumerate((which, other)):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(ids, *rounds[i][k])))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(p, q) for p, q in zip(outs, want[i]))
    s.sync()
    s.close()


def test_empty_batches():
    b = Batch(20, [3], [0], [2, 5], 12, 9, torch.float32)
    s = _server(b)
    ads = _adapters(s, b)
    none = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    for T in (0, 3):
        x, dy, base = b.x[:T].cuda(), b.dy[:T].cuda(), b.base[:T].cuda()
        out, shrunk = ads.forward(x, *none, base=base)
        assert torch.equal(out, base)
        ga, gb = ads.backward(x, dy, shrunk, *none)
        assert ga.shape == (7, 12) and gb.shape == (7, 9) and not ga.any() and not gb.any()
    s.sync()
    s.close()
