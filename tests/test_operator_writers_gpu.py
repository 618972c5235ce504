"""A call that writes rows waits for the operators that read them, or is refused: also while a
capture keeps the readers' stream from being asked."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError
from operator_refs import Batch

pytestmark = pytest.mark.gpu
A, B = 11, 12
UNSUPPORTED = 10


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.fixture(scope="module")
def hip():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as f:
        return ctypes.CDLL(next(ln.split()[-1] for ln in f if "libamdhip64" in ln))


def _case():
    b = Batch(41, [4000], [0], [64], 1024, 1024, torch.bfloat16)
    s = psa.Server(0, 1, [1])
    for t, w in ((A, b.a), (B, b.b)):
        s.CreateTable(t, psa.TableInfo(row_capacity=w.shape[1], max_rows=b.rows))
        s.load_rows(t, 0, w.numpy())
    ids = torch.tensor(b.begin, dtype=torch.int32).cuda(), torch.tensor(b.which, dtype=torch.int32).cuda()
    return b, s, s.create_adapters(A, B, b.adapters()), ids


def test_the_null_stream_behind_a_capture(hip):
    """Operators run on the null stream; while a blocking stream is captured that stream cannot be
    asked, so writers and sync are refused and change nothing; after it they wait as ever."""
    b, s, ads, ids = _case()
    x, base = b.x.cuda(), b.base.cuda()
    want = ads.forward(x, *ids, base=base)[0]
    rows = torch.arange(b.rows, dtype=torch.int32, device="cuda")
    big = torch.full((b.rows, 1024), 1e3, device="cuda")
    msg = s.pack_stream([dict(table_id=t, dtype=psa.F32, dense_serialized=True, row_ids=rows, oplogs=big) for t in (A, B)])
    s.sync()
    torch.cuda.synchronize()
    zero = np.zeros((b.rows, 1024), np.float32)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    outs = [torch.empty_like(base) for _ in range(4)]
    shrunk = torch.empty(ads.sizes(b.T)[0] // 4, device="cuda")
    for out in outs:
        ads.forward(x, *ids, base=base, out=out, shrunk=shrunk)
    assert hip.hipStreamBeginCapture(stream, 2) == 0   # relaxed
    got = []
    for call in (s.sync, lambda: s.load_rows(A, 0, zero), lambda: s.apply_device([(msg.data_ptr(), msg.numel(), 1, 0)]),
                 lambda: s.read_rows(A, 0, 1)):
        try:
            call()
            got.append(0)
        except PsxError as e:
            got.append(e.status)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert got == [UNSUPPORTED] * 4
    s.load_rows(A, 0, zero)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert torch.equal(ads.forward(x, *ids, base=base)[0], base)
    s.apply_device([(msg.data_ptr(), msg.numel(), 1, 0)])   # its version was not used up
    s.sync()
    assert bool((s.read_rows(A, 0, b.rows) == 1e3).all())
    assert hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0
    s.close()


def test_a_stream_under_capture_that_read_rows_before():
    b, s, ads, ids = _case()
    x, base = b.x.cuda(), b.base.cuda()
    side, out = torch.cuda.Stream(), torch.empty_like(base)
    shrunk = torch.empty(ads.sizes(b.T)[0] // 4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ads.forward(x, *ids, base=base, out=out, shrunk=shrunk)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ads.forward(x, *ids, base=base, out=out, shrunk=shrunk)
        with pytest.raises(PsxError) as e:
            s.load_rows(A, 0, np.zeros((b.rows, 1024), np.float32))
    assert e.value.status == UNSUPPORTED
    s.load_rows(A, 0, np.zeros((b.rows, 1024), np.float32))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, base)
    s.sync()
    s.close()
