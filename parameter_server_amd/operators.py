"""Operators on parameter rows that a context's tables hold (include/psx.h), over CUDA tensors.

Made by Server.create_adapters / checkpoint_store / position_bias.  Each call runs on torch's
current stream of the server's device, asynchronously; what only the GPU sees is reported by
Server.sync().  Wrong arguments raise PsxError before anything is launched.

None of them is an autograd function: outside torch.no_grad() (and an autograd.Function's own
forward and backward, where it holds) a tensor that requires a gradient is refused, since the
result would have none; gradients come from the backward() methods.  Checkpoints keep values alone.
"""
import ctypes

from . import _abi
from ._abi import PsxError, psx_adapter, psx_matrix, psx_requests, psx_scores

_INVALID = 1   # PSX_ERR_INVALID_ARG
_types = None


def _act(dtype, name):
    global _types
    if _types is None:
        import torch
        _types = {torch.float32: _abi.ACT_F32, torch.float16: _abi.ACT_F16, torch.bfloat16: _abi.ACT_BF16}
    t = _types.get(dtype)
    if t is None:
        raise PsxError(_INVALID, f"{name}: float32, float16 or bfloat16, not {dtype}")
    return t


def _on(server, t, name):
    if t.get_device() != server.device:   # -1 for a tensor on the host
        raise PsxError(_INVALID, f"{name}: not on the server's device")


def _matrix(server, t, name):
    if t.get_device() != server.device:
        _on(server, t, name)
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise PsxError(_INVALID, f"{name}: a 2-d tensor with consecutive columns")
    rows, cols = shape
    return psx_matrix(t.data_ptr(), _act(t.dtype, name), 0, rows, cols, stride[0] if rows > 1 else cols)


def _refuse_graph():
    """A tensor requires a gradient.  autograd would take the result for a constant, or for what was
    in the output's place."""
    import torch
    if torch.is_grad_enabled():
        raise PsxError(_INVALID, "a tensor requires a gradient, which this call does not record: use it under "
                                 "torch.no_grad() or within an autograd.Function, with the backward() methods")


def _stream(device):
    """The current stream's handle: a tenth of the time of torch.cuda.current_stream(), which a
    small call would notice."""
    import torch
    return torch._C._cuda_getCurrentRawStream(device)


class _Handle:
    """A handle that lives in a server's context."""

    def __init__(self, server, destroy):
        import torch
        self._server, self._destroy, self._h = server, destroy, ctypes.c_void_p()
        self._device = torch.device("cuda", server.device)

    def close(self):
        if self._h and self._server._ctx:   # a closed context has freed it
            getattr(self._server._L, self._destroy)(self._h)
        self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st):
        if st != _abi.PSX_OK:
            raise PsxError(st, self._server._L.psx_last_error(self._server._ctx).decode())

    def _live(self):
        if not self._h or not self._server._ctx:
            raise PsxError(_INVALID, "closed")
        return self._server._L

    def _stream(self):
        return _stream(self._server.device)

    def _empty(self, *shape):
        import torch
        return torch.empty(shape, dtype=torch.float32, device=self._device)


class AdapterSet(_Handle):
    """Low-rank adapters of many requests beside a shared projection (psx_adapters).

    num_rows: the ranks' sum; row_ids: CUDA int32 [num_rows], the rows that the gradients are
    increments of, in their order (as Server.pack_stream takes them)."""

    def __init__(self, server, table_a, table_b, adapters):
        import torch
        super().__init__(server, "psx_adapters_destroy")
        L = server._L
        arr = (psx_adapter * max(len(adapters), 1))(*[psx_adapter(int(f), int(r), float(s), 0) for f, r, s in adapters])
        self._check(L.psx_adapters_create(server._ctx, table_a, table_b, arr, len(adapters), ctypes.byref(self._h)))
        n = ctypes.c_int32()
        self._check(L.psx_adapters_info(self._h, ctypes.byref(n), None))
        self.num_rows = n.value
        self.widths = (server.tables[table_a].row_capacity, server.tables[table_b].row_capacity)
        step = server.tables[table_a].row_stride
        ids = [f + step * i for f, r, _ in adapters for i in range(r)]
        self.row_ids = torch.tensor(ids, dtype=torch.int32).to(torch.device("cuda", server.device))
        self._sizes = {}

    def sizes(self, num_tokens):
        """Bytes of (shrunk, work) for calls of num_tokens tokens."""
        got = self._sizes.get(num_tokens)
        if got is None:
            a, b = ctypes.c_size_t(), ctypes.c_size_t()
            self._check(self._live().psx_adapters_sizes(self._h, num_tokens, ctypes.byref(a), ctypes.byref(b)))
            if len(self._sizes) > 256:
                self._sizes.clear()
            got = self._sizes[num_tokens] = (a.value, b.value)
        return got

    def _requests(self, begin, adapter):
        import torch
        for t, name in ((begin, "request_begin"), (adapter, "request_adapter")):
            if t.get_device() != self._server.device:
                _on(self._server, t, name)
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise PsxError(_INVALID, f"{name}: a contiguous 1-d int32 tensor")
        n = adapter.shape[0]
        if begin.shape[0] != n + 1:
            raise PsxError(_INVALID, "request_begin has one entry more than request_adapter")
        return psx_requests(begin.data_ptr(), adapter.data_ptr(), n, 0)

    def _buffer(self, t, nbytes, name):
        if t is None:
            return self._empty(nbytes // 4)
        _on(self._server, t, name)
        if not t.is_contiguous() or t.numel() * t.element_size() < nbytes:
            raise PsxError(_INVALID, f"{name}: {nbytes} contiguous bytes")
        return t

    def forward(self, x, request_begin, request_adapter, base=None, out=None, shrunk=None):
        """out = base + scale (x A^T) B for every request's tokens; returns (out, shrunk).

        x [tokens, width of A], base and out [tokens, width of B], of one type.  out may be base.
        Rows of out outside all requests stay as they were; without out, a copy of base (or
        zeros) takes its place.  shrunk (made here, or a buffer of sizes()[0] bytes) is what
        backward() of the same tokens reads."""
        import torch
        L = self._live()
        if x.requires_grad or (base is not None and base.requires_grad) or (out is not None and out.requires_grad):
            _refuse_graph()
        xm = _matrix(self._server, x, "x")
        bm = _matrix(self._server, base, "base") if base is not None else None
        written = [t for t in (out, shrunk) if t is not None]
        if out is None:
            out = (base.clone(memory_format=torch.contiguous_format) if base is not None
                   else torch.zeros(x.shape[0], self.widths[1], dtype=x.dtype, device=x.device))
        om = _matrix(self._server, out, "out")
        r = self._requests(request_begin, request_adapter)
        shrunk = self._buffer(shrunk, self.sizes(x.shape[0])[0], "shrunk")
        self._check(L.psx_adapters_forward(self._h, r, xm, bm, om, shrunk.data_ptr(), self._stream()))
        if written:   # autograd has to see it if a graph has kept one of them
            torch.autograd.graph.increment_version(written)
        return out, shrunk

    def backward(self, x, dy, shrunk, request_begin, request_adapter, base=None, out=None, scale=1.0, grad_a=None,
                 grad_b=None, work=None):
        """Gradients times `scale` of that forward call's rows: (grad_a, grad_b), f32 [num_rows,
        width], rows as in row_ids.  x: the forward call's, or its Checkpoint.  With out (and base):
        out = base + scale_of_adapter (dy B^T) A, the gradient of x."""
        import torch
        L = self._live()
        if dy.requires_grad or (base is not None and base.requires_grad):
            _refuse_graph()
        written = [t for t in (out, grad_a, grad_b) if t is not None]
        for t in written:
            if t.requires_grad:
                _refuse_graph()
        if isinstance(x, Checkpoint):
            if (x.rows, x.cols) != (dy.shape[0], self.widths[0]):
                raise PsxError(_INVALID, "x: a checkpoint of another shape")
            _on(self._server, x.buffer, "x")
            xm, ck = None, x.buffer.data_ptr()
        else:
            if x.requires_grad:
                _refuse_graph()
            xm, ck = _matrix(self._server, x, "x"), None
        dm = _matrix(self._server, dy, "dy")
        om = _matrix(self._server, out, "out") if out is not None else None
        bm = _matrix(self._server, base, "base") if base is not None else None
        r = self._requests(request_begin, request_adapter)
        need = self.sizes(dy.shape[0])
        _on(self._server, shrunk, "shrunk")
        shrunk = self._buffer(shrunk, need[0], "shrunk")
        work = self._buffer(work, need[1], "work")
        grads = []
        for g, width, name in ((grad_a, self.widths[0], "grad_a"), (grad_b, self.widths[1], "grad_b")):
            if g is None:
                grads.append(self._empty(self.num_rows, width))
                continue
            _on(self._server, g, name)
            if g.dtype != torch.float32 or tuple(g.shape) != (self.num_rows, width) or not g.is_contiguous():
                raise PsxError(_INVALID, f"{name}: contiguous float32 [num_rows, width]")
            grads.append(g)
        self._check(L.psx_adapters_backward(self._h, r, xm, ck, dm, shrunk.data_ptr(), bm, om, grads[0].data_ptr(),
                                            grads[1].data_ptr(), float(scale), work.data_ptr(), self._stream()))
        if written:   # autograd has to see it if a graph has kept one of them
            torch.autograd.graph.increment_version(written)
        return grads[0], grads[1]


class Checkpoint:
    """A 2-d activation kept in 8 bits (psx_checkpoint_store): .buffer uint8, .rows, .cols, .dtype."""

    def __init__(self, server, x):
        import torch
        self._server = server
        m = _matrix(server, x, "x")
        self.rows, self.cols, self.dtype = m.rows, m.cols, x.dtype
        n = ctypes.c_size_t()
        st = server._L.psx_checkpoint_bytes(m.rows, m.cols, ctypes.byref(n))
        if st != _abi.PSX_OK:
            raise PsxError(st, "bad shape")
        self.buffer = torch.empty(n.value, dtype=torch.uint8, device=x.device)
        self._call("psx_checkpoint_store", m, self.buffer.data_ptr())

    def _call(self, name, a, b):
        srv = self._server
        if not srv._ctx:
            raise PsxError(_INVALID, "closed")
        st = getattr(srv._L, name)(srv._ctx, a, b, _stream(srv.device))
        if st != _abi.PSX_OK:
            raise PsxError(st, srv._L.psx_last_error(srv._ctx).decode())

    def load(self, dtype=None, out=None):
        """The stored values, in dtype (default: the activation's) or into out."""
        import torch
        given = out is not None
        if given:
            if out.requires_grad:
                _refuse_graph()
        else:
            out = torch.empty(self.rows, self.cols, dtype=dtype or self.dtype, device=self.buffer.device)
        m = _matrix(self._server, out, "out")
        if (m.rows, m.cols) != (self.rows, self.cols):
            raise PsxError(_INVALID, "out: another shape")
        self._call("psx_checkpoint_load", self.buffer.data_ptr(), m)
        if given:
            torch.autograd.graph.increment_version((out,))   # autograd has to see it if a graph has kept it
        return out


class PositionBias(_Handle):
    """A learned relative position bias by buckets (psx_position_bias)."""

    def __init__(self, server, table_id, first_row, num_buckets, max_distance, bidirectional):
        super().__init__(server, "psx_position_bias_destroy")
        self._check(server._L.psx_position_bias_create(server._ctx, table_id, first_row, num_buckets, max_distance,
                                                       1 if bidirectional else 0, ctypes.byref(self._h)))
        self.num_buckets, self.heads = num_buckets, server.tables[table_id].row_capacity

    def _scores(self, t, name):
        if t.get_device() != self._server.device:
            _on(self._server, t, name)
        shape, stride = t.shape, t.stride()
        if len(shape) == 3:
            shape, stride = (1, *shape), (0, *stride)
        if len(shape) != 4 or (shape[3] > 1 and stride[3] != 1):
            raise PsxError(_INVALID, f"{name}: [batch, heads, queries, keys] with consecutive keys")
        b, h, q, k = shape
        # strides of axes with one entry say nothing
        return psx_scores(t.data_ptr(), _act(t.dtype, name), 0, b, h, q, k, stride[0] if b > 1 else 0,
                          stride[1] if h > 1 else 0, stride[2] if q > 1 else k)

    def forward(self, q_len, k_len, q_begin=0, dtype=None, out=None):
        """The bias of queries at positions q_begin .. q_begin + q_len against keys 0 .. k_len:
        [heads, q_len, k_len] in dtype (default float32), or into out."""
        import torch
        L = self._live()
        given = out is not None
        if not given:
            out = torch.empty(self.heads, q_len, k_len, dtype=dtype or torch.float32, device=self._device)
        elif out.dim() != 3 or tuple(out.shape) != (self.heads, q_len, k_len):
            raise PsxError(_INVALID, "out: [heads, q_len, k_len]")
        elif out.requires_grad:
            _refuse_graph()
        self._check(L.psx_position_bias_forward(self._h, self._scores(out, "out"), q_begin, self._stream()))
        if given:
            torch.autograd.graph.increment_version((out,))   # autograd has to see it if a graph has kept it
        return out

    def backward(self, d, q_begin=0, scale=1.0, grad=None, work=None):
        """scale times the gradient of the bucket rows, f32 [num_buckets, heads], from d
        [batch, heads, queries, keys] (or one batch entry)."""
        import torch
        L = self._live()
        if d.requires_grad:
            _refuse_graph()
        s = self._scores(d, "d")
        n = ctypes.c_size_t()
        self._check(L.psx_position_bias_work(self._h, s.batch, s.q_len, s.k_len, ctypes.byref(n)))
        if work is None:
            work = self._empty(n.value // 4)
        else:
            _on(self._server, work, "work")
            if not work.is_contiguous() or work.numel() * work.element_size() < n.value:
                raise PsxError(_INVALID, f"work: {n.value} contiguous bytes")
        given = grad is not None
        if not given:
            grad = self._empty(self.num_buckets, self.heads)
        else:
            if grad.requires_grad:
                _refuse_graph()
            _on(self._server, grad, "grad")
            if (grad.dtype != torch.float32 or tuple(grad.shape) != (self.num_buckets, self.heads)
                    or not grad.is_contiguous()):
                raise PsxError(_INVALID, "grad: contiguous float32 [num_buckets, heads]")
        self._check(L.psx_position_bias_backward(self._h, s, q_begin, float(scale), grad.data_ptr(), work.data_ptr(),
                                                 self._stream()))
        if given:
            torch.autograd.graph.increment_version((grad,))   # autograd has to see it if a graph has kept it
        return grad
