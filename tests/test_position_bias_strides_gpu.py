"""Position bias: every layout whose values lie within reach is taken, whatever its strides; what
does not fit a launch is refused before one."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import numpy as np

import parameter_server_amd as psa
from parameter_server_amd import _abi
from operator_refs import bucket, buckets_of, off

pytestmark = pytest.mark.gpu
TABLE, BUCKETS, DISTANCE = 5, 8, 20


@pytest.fixture(scope="module", autouse=True)
def _gpu(built_lib):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _bias(heads):
    s = psa.Server(0, 1)
    s.CreateTable(TABLE, psa.TableInfo(row_capacity=heads, max_rows=BUCKETS))
    w = np.random.RandomState(heads).normal(size=(BUCKETS, heads)).astype(np.float32)
    s.load_rows(TABLE, 0, w)
    return s, torch.from_numpy(w), s.position_bias(TABLE, 0, BUCKETS, DISTANCE, True)


def _line(k, begin):
    """Buckets of one query against k keys."""
    near = range(max(0, begin - 40), min(k, begin + 41))
    at = torch.empty(k, dtype=torch.long)
    at[:begin] = bucket(-DISTANCE, BUCKETS, DISTANCE, True)
    at[begin:] = bucket(DISTANCE, BUCKETS, DISTANCE, True)
    for i in near:
        at[i] = bucket(i - begin, BUCKETS, DISTANCE, True)
    return at


@pytest.mark.parametrize("q", [1, 2])
def test_more_than_2_to_22_keys(q):
    k, begin = (1 << 22) + 5, 1 << 21
    s, w, bias = _bias(2)
    got = bias.forward(q, k, begin, torch.bfloat16).cpu()
    at = torch.stack([_line(k, begin + i) for i in range(q)])
    assert torch.equal(got, w.t()[:, at].bfloat16())
    d = torch.ones(1, 2, q, k, dtype=torch.bfloat16, device="cuda")
    grad = bias.backward(d, begin, 0.5).cpu().double()
    counts = torch.bincount(at.flatten(), minlength=BUCKETS).double()
    # sums of ones: whole numbers below 2^24 are exact in f32, above them half a step
    assert bool(((grad - 0.5 * counts[:, None]).abs() <= 2.0 ** -24 * counts[:, None]).all())
    s.close()


def test_queries_over_heads_of_a_long_context():
    """[query][head][key] with 64 heads x 131072 keys: a query's stride is 2^23."""
    heads, q, k = 64, 3, 131072
    s, w, bias = _bias(heads)
    buf = torch.empty(q, heads, k, dtype=torch.bfloat16, device="cuda")
    bias.forward(q, k, k - q, out=buf.transpose(0, 1))
    at = torch.stack([_line(k, k - q + i) for i in range(q)])
    assert torch.equal(buf.transpose(0, 1).cpu(), w.t()[:, at].bfloat16())
    d = torch.ones(2, q, heads, k, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    grad = bias.backward(d, k - q).cpu().double()
    counts = 2 * torch.bincount(at.flatten(), minlength=BUCKETS).double()
    assert bool(((grad - counts[:, None]).abs() <= 2.0 ** -24 * counts[:, None]).all())
    s.close()


def test_axes_of_one_entry_have_no_stride():
    s, w, bias = _bias(3)
    m = torch.randn(1, 3, 6, 7, device="cuda")
    far = _abi.psx_scores(m.data_ptr(), 0, 0, 1, 3, 6, 7, 1 << 60, 42, 7)   # the batch's
    grad, work = torch.zeros(BUCKETS, 3, device="cuda"), torch.zeros(1 << 16, device="cuda")
    assert s._L.psx_position_bias_backward(bias._h, ctypes.byref(far), 0, 1.0, grad.data_ptr(), work.data_ptr(), None) == 0
    hot = torch.nn.functional.one_hot(buckets_of(6, 7, 0, BUCKETS, DISTANCE, True).flatten(), BUCKETS).double()
    flat = m[0].double().cpu().reshape(3, -1)
    assert off(grad, (flat @ hot).t(), 128 * 2.0 ** -24 * (flat.abs() @ hot).t() + 1e-40) <= 1
    one = torch.full((3, 1, 7), 9.0, device="cuda")
    out = _abi.psx_scores(one.data_ptr(), 0, 0, 1, 3, 1, 7, 0, 7, 1 << 60)   # the query's
    assert s._L.psx_position_bias_forward(bias._h, ctypes.byref(out), 0, None) == 0
    assert torch.equal(one.cpu(), w.t()[:, buckets_of(1, 7, 0, BUCKETS, DISTANCE, True)])
    s.close()


@pytest.mark.parametrize("name,scores", [
    ("forward", (1, 2, 1 << 24, 1 << 20, 0, 1 << 45, 1 << 23)),    # rows reach past 2^46
    ("forward", (1, 2, 16, 64, 0, (1 << 46) + 1, 64)),
    ("backward", (65535, 2, 16, 64, 1 << 46, 1024, 64)),
    ("backward", (2, 2, 16, 64, 0, 0, -1)),
    ("backward", (2, 2, 16, 64, -1, 0, 64)),
    ("backward", (2, 2, 16, 64, 1 << 62, 1 << 62, 1 << 62)),
])
def test_strides_past_reach_are_refused(name, scores):
    s, _, bias = _bias(2)
    m = torch.zeros(64, device="cuda")
    c = _abi.psx_scores(m.data_ptr(), 0, 0, *scores)
    if name == "forward":
        st = s._L.psx_position_bias_forward(bias._h, ctypes.byref(c), 0, None)
    else:
        st = s._L.psx_position_bias_backward(bias._h, ctypes.byref(c), 0, 1.0, m.data_ptr(), m.data_ptr(), None)
    assert st == 1
    s.close()


def test_more_scores_than_a_launch_has_blocks_are_refused():
    s, _, bias = _bias(2)
    m = torch.zeros(64, device="cuda")
    # 2^22 x 2^24: within reach of the strides, 2^29 blocks
    c = _abi.psx_scores(m.data_ptr(), 2, 0, 1, 2, 1 << 22, 1 << 24, 0, 1 << 46, 1 << 24)
    assert s._L.psx_position_bias_forward(bias._h, ctypes.byref(c), 0, None) == 10
    s.close()
