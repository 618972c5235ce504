"""Activations kept in 8 bits against a restatement in 64 bits: what reads back is equal bit for
bit (every step of the definition is exact but the one rounding to an integer)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import parameter_server_amd as psa
from parameter_server_amd import PsxError, _abi
from operator_refs import checkpoint

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def srv(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    s = psa.Server(0, 1)
    yield s
    s.close()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 1001), (70, 8), (4, 2050), (4099, 3)])
def test_round_trip(srv, dt, rows, cols):
    g = torch.Generator().manual_seed(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dt)
    x[0, 0] = 0
    x[-1] = 0
    ck = srv.checkpoint_store(x.cuda())
    want = checkpoint(x)
    for out in DT:
        got = ck.load(out).cpu()
        fits = want.to(torch.float32).clamp(-torch.finfo(out).max, torch.finfo(out).max).to(out)   # NaN stays NaN
        assert got.dtype == out and bool(((got == fits) | (torch.isnan(got) & torch.isnan(fits))).all())
    assert ck.load().dtype == dt
    step = (ck.load(torch.float32).cpu().double() - x.double()).abs()
    pad = torch.nn.functional.pad(x.double().abs(), (0, -cols % 32)).reshape(rows, -1, 32).amax(2)
    inside = torch.isfinite(pad).repeat_interleave(32, 1)[:, :cols]   # binary16 overflows for some rows
    assert bool((step[inside] <= (pad / 127).repeat_interleave(32, 1)[:, :cols][inside] + 2.0 ** -127).all())   # 2^e < 2 max / 127, half of it


def test_bytes(srv):
    """Codes, then exponents, as documented; zero codes behind a row's last value."""
    x = torch.tensor([[1.0, -2.0, 127.0, 0.4], [0.0, 0.0, 0.0, 0.0], [254.5, 1.0, 3.0, -1.0]]).cuda()
    b = srv.checkpoint_store(x).buffer.cpu()
    assert b.numel() == 3 * 33
    codes = b[:96].view(torch.int8).reshape(3, 32)
    assert codes[0, :4].tolist() == [1, -2, 127, 0] and codes[1].abs().sum() == 0
    assert codes[2, :4].tolist() == [64, 0, 1, 0]   # ties to even: 0.25, 0.75, -0.25 steps of 4
    assert codes[:, 4:].abs().sum() == 0
    assert b[96:].tolist() == [127, 1, 129]


@pytest.mark.parametrize("dt", DT)
def test_extremes(srv, dt):
    """Borders of the exponent, the largest values, subnormals, ties, and groups that are not finite."""
    big = torch.finfo(dt).max
    rows = [[big, 1.0, -big / 2], [127.0, 63.5, 0.5], [127.5, 1.5, -2.5], [128.0, 3.0, 1.0], [254.0, 255.0, 1.0],
            [float(torch.finfo(dt).tiny), -float(torch.finfo(dt).smallest_normal) / 2, 0.0], [1e-7, 1e-7, -3e-8]]
    x = torch.zeros(len(rows), 40, dtype=dt)
    for i, r in enumerate(rows):
        x[i, 30:33] = torch.tensor(r).to(dt)   # two groups a row
    ck = srv.checkpoint_store(x.cuda())
    want = checkpoint(x)
    assert torch.equal(ck.load(torch.float32).cpu().double(), want)
    half = ck.load(torch.float16).cpu()
    assert bool(torch.isfinite(half).all())
    assert torch.equal(half, want.float().clamp(-65504, 65504).half())
    y = torch.ones(3, 70, dtype=dt)
    y[0, 3] = float("inf")
    y[1, 40] = float("nan")
    y[2, 69] = -float("inf")
    got = srv.checkpoint_store(y.cuda()).load().cpu()
    bad = torch.zeros(3, 70, dtype=torch.bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 64:] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], y[~bad])


@pytest.mark.parametrize("dt", DT)
def test_strides(srv, dt):
    """Rows at odd addresses and apart from one another; what lies between stays."""
    buf = torch.randn(9, 77, generator=torch.Generator().manual_seed(2)).to(dt).cuda()
    x = buf[1:8, 3:68]
    ck = srv.checkpoint_store(x)
    out = torch.full_like(buf, 5.0)
    assert ck.load(out=out[1:8, 3:68]).data_ptr() == out[1:8, 3:68].data_ptr()
    full = torch.full_like(buf, 5.0).cpu()
    full[1:8, 3:68] = checkpoint(x.cpu()).to(dt)
    assert torch.equal(out.cpu(), full)
    one = srv.checkpoint_store(buf[:1, :50].expand(6, 50)).load()   # a broadcast row
    assert torch.equal(one, srv.checkpoint_store(buf[:1, :50]).load().expand(6, 50))


def test_empty_and_refusals(srv):
    for shape in [(0, 5), (5, 0), (0, 0)]:
        assert srv.checkpoint_store(torch.zeros(shape, device="cuda")).load().shape == shape
    x = torch.zeros(4, 64, device="cuda")
    for bad in [x.cpu(), x.double(), x[0], x.t(), x[:, ::2]]:
        with pytest.raises(PsxError) as e:
            srv.checkpoint_store(bad)
        assert e.value.status == 1
    ck = srv.checkpoint_store(x)
    for bad in [x[:3], x[:, :63], x[:1].expand(4, 64)]:
        with pytest.raises(PsxError) as e:
            ck.load(out=bad)
        assert e.value.status == 1


def test_on_a_stream_and_in_a_graph(srv):
    x = torch.randn(64, 300, device="cuda").bfloat16()
    want = checkpoint(x.cpu()).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = srv.checkpoint_store(x).load()
    side.synchronize()
    assert torch.equal(got.cpu(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = srv.checkpoint_store(x).load()
    for seed in range(3):
        x.copy_(torch.randn(64, 300, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), checkpoint(x.cpu()).bfloat16())
        assert torch.equal(srv.checkpoint_store(x).load(), y)


def test_rows_past_a_launch_are_refused(srv):
    x = torch.zeros(4, device="cuda")
    for cols in ((1 << 30) + 1, 1 << 40):
        m = _abi.psx_matrix(x.data_ptr(), 0, 0, 1, cols, cols)
        for name, args in (("psx_checkpoint_store", (ctypes.byref(m), 4096)), ("psx_checkpoint_load", (4096, ctypes.byref(m)))):
            assert getattr(srv._L, name)(srv._ctx, *args, None) == 10
