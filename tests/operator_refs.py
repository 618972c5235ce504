"""64-bit references of the operators on parameter rows, and what they may be off by."""
import numpy as np
import torch

F23 = 2.0 ** -23   # a sum of n f32 terms, in any order and with any rounding, is off by n * 2^-23 of the terms' magnitudes
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half a step of binary16's subnormals


def off(got, want, tol):
    """Worst of |got - want| / tol (inf where one is finite and the other not)."""
    got, want = got.double().cpu(), want.double().cpu()
    tol = tol.double().cpu() if torch.is_tensor(tol) else torch.full_like(want, tol)
    d = (got - want).abs()
    d = torch.where(torch.isfinite(d), d, torch.full_like(d, float("inf")))
    return float((d / tol.clamp(min=1e-300)).max()) if d.numel() else 0.0


class Batch:
    """Requests over two tables of adapter rows, all tensors on the CPU in 64 bits where it matters."""

    def __init__(self, seed, lengths, which, ranks, d_in, d_out, dtype, lead=0, tail=0, gap_rows=1, x_pad=0, scales=None):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.which, self.ranks, self.dtype = lengths, which, ranks, dtype
        self.d_in, self.d_out = d_in, d_out
        self.begin = lead + np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
        self.T = int(self.begin[-1]) + tail
        self.first, at = [], 3   # rows no adapter owns in front of and between the adapters
        for r in ranks:
            self.first.append(at)
            at += r + gap_rows
        self.rows = at + 2
        self.scales = scales or [0.5 + 0.25 * i for i in range(len(ranks))]
        self.a = torch.randn(self.rows, d_in, generator=g) * d_in ** -0.5
        self.b = torch.randn(self.rows, d_out, generator=g) * 0.1

        def act(cols):
            return torch.randn(self.T, cols + x_pad, generator=g).to(dtype)[:, :cols]

        self.x, self.base, self.dy, self.dbase = act(d_in), act(d_out), act(d_out), act(d_in)

    def adapters(self):
        return list(zip(self.first, self.ranks, self.scales))

    def segments(self):
        for n, i in enumerate(self.which):
            yield slice(int(self.begin[n]), int(self.begin[n + 1])), i

    def rows_of(self, i):
        return slice(self.first[i], self.first[i] + self.ranks[i])

    def forward(self, out, base=True):
        """(out, tolerance): `out` where no request has the token."""
        want, tol = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64)
        two = 0.0 if self.dtype == torch.float32 else 2.0 ** -15   # expand: two parts a factor
        for at, i in self.segments():
            b0 = self.base[at].double() if base else torch.zeros(at.stop - at.start, self.d_out, dtype=torch.float64)
            want[at] = b0
            if i >= 0:
                a, b = self.a[self.rows_of(i)].double(), self.b[self.rows_of(i)].double()
                x, s = self.x[at].double(), self.scales[i]
                want[at] += s * (x @ a.t()) @ b
                mag = abs(s) * (x.abs() @ a.abs().t()) @ b.abs()
                tol[at] += ((self.d_in + self.ranks[i] + 16) * F23 + two) * mag + F23 * (b0.abs() + mag)
            tol[at] += ROUND[self.dtype] * (want[at].abs() + tol[at]) + TINY[self.dtype]
        return want, tol

    def backward(self, out, gain, x=None, base=True):
        """({dx, grad_a, grad_b}, tolerances); x: the activation that the gradient of A uses."""
        x_used = (self.x if x is None else x).double()
        dx, dx_tol = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64)
        n = sum(self.ranks)
        grads = {k: torch.zeros(n, w, dtype=torch.float64) for k, w in (("a", self.d_in), ("b", self.d_out))}
        mags = {k: torch.zeros_like(v) for k, v in grads.items()}
        two = 0.0 if self.dtype == torch.float32 else 2.0 ** -15
        for at, i in self.segments():
            b0 = self.dbase[at].double() if base else torch.zeros(at.stop - at.start, self.d_in, dtype=torch.float64)
            dx[at] = b0
            if i >= 0:
                a, b, s = self.a[self.rows_of(i)].double(), self.b[self.rows_of(i)].double(), self.scales[i]
                x, dy = self.x[at].double(), self.dy[at].double()
                u, um = s * dy @ b.t(), abs(s) * dy.abs() @ b.abs().t()
                v, vm = s * x @ a.t(), abs(s) * x.abs() @ a.abs().t()
                dx[at] += u @ a
                mag = um @ a.abs()
                dx_tol[at] += ((self.d_out + self.ranks[i] + 16) * F23 + two) * mag + F23 * (b0.abs() + mag)
                o = sum(self.ranks[:i])
                rows = slice(o, o + self.ranks[i])
                grads["a"][rows] += gain * u.t() @ x_used[at]
                mags["a"][rows] += abs(gain) * um.t() @ x_used[at].abs()
                grads["b"][rows] += gain * v.t() @ dy
                mags["b"][rows] += abs(gain) * vm.t() @ dy.abs()
            dx_tol[at] += ROUND[self.dtype] * (dx[at].abs() + dx_tol[at]) + TINY[self.dtype]
        ta = (self.T + self.d_out + 64) * F23 * mags["a"]
        tb = (self.T + self.d_in + 64) * F23 * mags["b"]
        return {"dx": dx, "grad_a": grads["a"], "grad_b": grads["b"]}, {"dx": dx_tol, "grad_a": ta, "grad_b": tb}


def checkpoint(x):
    """The values that an 8-bit checkpoint of x [rows, cols] stands for, in 64 bits."""
    v = np.asarray(x.double())
    rows, cols = v.shape
    p = np.zeros((rows, -(-cols // 32) * 32))
    p[:, :cols] = v
    p = p.reshape(rows, -1, 32)
    out = np.zeros_like(p)
    for r in range(rows):
        for g in range(p.shape[1]):
            top = np.abs(p[r, g]).max()
            if not np.isfinite(top):
                out[r, g] = np.nan
                continue
            e = -126
            while e < 122 and 127 * 2.0 ** e < top:
                e += 1
            most = 63 if e == 122 else 127
            out[r, g] = np.clip(np.rint(p[r, g] / 2.0 ** e), -most, most) * 2.0 ** e
    return torch.from_numpy(out.reshape(rows, -1)[:, :cols].copy())


def bucket(r, buckets, distance, both):
    """The bucket of a relative position, by whole numbers."""
    half = buckets // 2 if both else buckets
    n = abs(r) if both else max(-r, 0)
    exact = half // 2
    m = half - exact
    b = n
    if n >= exact:
        n = min(n, distance)
        b = exact + sum(1 for i in range(1, m) if n ** m * exact ** i >= distance ** i * exact ** m)
    return b + (half if both and r > 0 else 0)


def buckets_of(q, k, begin, buckets, distance, both):
    """[q, k] of bucket numbers."""
    line = np.array([bucket(r, buckets, distance, both) for r in range(-(q - 1) - begin, k - begin)], dtype=np.int64)
    at = np.arange(k)[None, :] - np.arange(q)[:, None] + (q - 1)
    return torch.from_numpy(line[at])
