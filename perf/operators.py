"""The operators on parameter rows, as workloads: what each takes, its plain form, its work.

    adapters    low-rank adapters of many requests beside a shared projection: the rank rows are rows
                of two tables; forward (serving and training) and backward (row increments)
    checkpoint  an activation kept in 8 bits: stored and loaded again
    bias        a learned relative position bias by buckets whose rows are a table's, and its gradient

`own` selects the framework's calls; otherwise run() is elementary torch in 32 bits.
"""
import math
import random

import torch

own = False

TABLE_A, TABLE_B, TABLE_BIAS = 1, 2, 3
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------------


def listed():
    return [
        # a decode step: eight requests, one token each, every one with its own adapter
        {"name": "adapters_decode", "op": "adapters", "backward": False, "dtype": "bf16", "d_in": 2048, "d_out": 2048,
         "tokens": 8, "requests": 8, "adapters": 8, "ranks": "16", "none": 0, "pad": 0, "checkpoint": False},
        # a serving step of prompts and single tokens together, adapters of several ranks, requests
        # without one, odd widths and a padded tail
        {"name": "adapters_mixed", "op": "adapters", "backward": False, "dtype": "f16", "d_in": 2047, "d_out": 4095,
         "tokens": 1531, "requests": 61, "adapters": 24, "ranks": "8,16,32,64", "none": 7, "pad": 5, "checkpoint": False},
        # the forward pass of a training batch: sixteen sequences, eight adapters
        {"name": "adapters_batch", "op": "adapters", "backward": False, "dtype": "bf16", "d_in": 4096, "d_out": 4096,
         "tokens": 16384, "requests": 16, "adapters": 8, "ranks": "16", "none": 0, "pad": 0, "checkpoint": False},
        # a small model in 32 bits: odd widths, uneven ranks
        {"name": "adapters_backward_small", "op": "adapters", "backward": True, "dtype": "f32", "d_in": 513, "d_out": 1025,
         "tokens": 77, "requests": 3, "adapters": 2, "ranks": "5,12", "none": 0, "pad": 2, "checkpoint": False},
        # the backward pass of a batch, from the activation as it was
        {"name": "adapters_backward", "op": "adapters", "backward": True, "dtype": "bf16", "d_in": 4096, "d_out": 4096,
         "tokens": 4096, "requests": 8, "adapters": 4, "ranks": "32", "none": 0, "pad": 0, "checkpoint": False},
        # the backward pass of a long batch, from the activation's 8-bit checkpoint
        {"name": "adapters_backward_checkpoint", "op": "adapters", "backward": True, "dtype": "bf16", "d_in": 4096,
         "d_out": 8192, "tokens": 16384, "requests": 16, "adapters": 4, "ranks": "64", "none": 0, "pad": 0,
         "checkpoint": True},
        # a small activation of odd width kept in 8 bits
        {"name": "checkpoint_small", "op": "checkpoint", "dtype": "f16", "rows": 129, "cols": 1001},
        # a layer's activation of a long batch
        {"name": "checkpoint_large", "op": "checkpoint", "dtype": "bf16", "rows": 16384, "cols": 8192},
        # one new token against a long context
        {"name": "bias_decode", "op": "bias", "backward": False, "dtype": "f32", "heads": 32, "q": 1, "k": 8191, "batch": 1,
         "buckets": 32, "distance": 128, "both": False},
        # a whole prompt
        {"name": "bias_prompt", "op": "bias", "backward": False, "dtype": "bf16", "heads": 32, "q": 2048, "k": 2048,
         "batch": 1, "buckets": 32, "distance": 128, "both": True},
        # the gradient of a small batch in 32 bits, odd lengths
        {"name": "bias_gradient_small", "op": "bias", "backward": True, "dtype": "f32", "heads": 12, "q": 77, "k": 131,
         "batch": 2, "buckets": 32, "distance": 128, "both": False},
        # the gradient of a training batch: the bias is shared by its sequences
        {"name": "bias_gradient", "op": "bias", "backward": True, "dtype": "bf16", "heads": 16, "q": 2048, "k": 2048,
         "batch": 4, "buckets": 32, "distance": 128, "both": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["adapters", "adapters", "adapters", "checkpoint", "bias", "bias"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "adapters":
        wide = [_log_int(rng, 64, 8192) for _ in range(2)]
        if rng.random() < 0.6:
            wide = [max(64, w // 64 * 64) for w in wide]
        tokens = min(_log_int(rng, 1, 16384), (1 << 27) // (sum(wide) * SIZES[dtype] // 2))
        requests = min(tokens, _log_int(rng, 1, 64))
        ranks = rng.choice(["16", "8", "64", "5,12", "8,16,32,64", "1,7,33"])
        backward = rng.random() < 0.5
        return {"op": op, "backward": backward, "dtype": dtype, "d_in": wide[0], "d_out": wide[1], "tokens": tokens,
                "requests": requests, "adapters": rng.randint(1, 12), "ranks": ranks, "none": requests // 8,
                "pad": rng.randint(0, 9), "checkpoint": backward and rng.random() < 0.5}
    if op == "checkpoint":
        cols = _log_int(rng, 1, 16384)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        return {"op": op, "dtype": dtype, "rows": min(_log_int(rng, 1, 16384), (1 << 28) // (cols * SIZES[dtype])),
                "cols": cols}
    q, k = _log_int(rng, 1, 4096), _log_int(rng, 1, 8192)
    if rng.random() < 0.5:
        k = max(8, k // 8 * 8)
    heads = rng.randint(1, 32)
    backward = rng.random() < 0.5
    batch = rng.randint(1, 4) if backward else 1
    room = (1 << 28) // SIZES[dtype]
    heads = max(1, min(heads, room // (q * k * batch)))
    buckets = rng.choice([8, 32, 32, 64])
    return {"op": op, "backward": backward, "dtype": dtype, "heads": heads, "q": q, "k": k, "batch": batch,
            "buckets": buckets, "distance": rng.choice([128, 128, 100, 513]), "both": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------


def _adapter_ranks(case):
    kinds = [int(r) for r in case["ranks"].split(",")]
    return [kinds[i % len(kinds)] for i in range(case["adapters"])]


def _adapter_inputs(case, seed):
    """Tensors of a batch of requests, on the GPU."""
    rng = random.Random(seed * 7919 + 17)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, N, pad = case["tokens"], case["requests"], case["pad"]
    dt = DTYPES[case["dtype"]]
    cuts = list(range(T + 1)) if N == T else [0] + sorted(rng.choices(range(T + 1), k=N - 1)) + [T]   # some are empty
    which = [rng.randrange(case["adapters"]) for _ in range(N)]
    which = [-1 if n < case["none"] else a for n, a in enumerate(which)]
    rng.shuffle(which)
    ranks = _adapter_ranks(case)
    rows = sum(ranks)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = {"ranks": ranks, "scales": [2.0 * 16 / (16 + r) for r in ranks],
         "begin": torch.tensor(cuts, dtype=torch.int32).cuda(), "which": torch.tensor(which, dtype=torch.int32).cuda(),
         "a": normal(rows, case["d_in"], std=case["d_in"] ** -0.5), "b": normal(rows, case["d_out"], std=0.02),
         "x": normal(T + pad, case["d_in"]).to(dt)}
    if case["backward"]:
        s["dy"] = normal(T + pad, case["d_out"], std=1e-3).to(dt)
        s["base"] = normal(T + pad, case["d_in"], std=1e-3).to(dt)
        s["gain"] = -0.01
    else:
        s["base"] = normal(T + pad, case["d_out"]).to(dt)
    return s


def _bias_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"w": torch.randn(case["buckets"], case["heads"], generator=g, device="cuda"),
         "begin": max(0, case["k"] - case["q"])}
    if case["backward"]:
        shape = (case["batch"], case["heads"], case["q"], case["k"])
        s["d"] = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(0.0, 1e-2, generator=g)
        s["gain"] = -0.01
    return s


def _activation(case, seed):
    """A residual stream's values: a few columns stand far out, some groups are zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(case["rows"], case["cols"], generator=g, device="cuda")
    far = torch.rand(case["cols"], generator=g, device="cuda") < 0.01
    x = torch.where(far, x * 40, x)
    x[:, : min(32, case["cols"])] *= (torch.rand(case["rows"], 1, generator=g, device="cuda") < 0.9)
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    if case["op"] == "checkpoint":
        s = {"x": _activation(case, seed)}
    elif case["op"] == "bias":
        s = _bias_inputs(case, seed)
    else:
        s = _adapter_inputs(case, seed)
    s["case"] = case
    if own:
        import parameter_server_amd as psa

        s["server"] = srv = psa.Server(torch.cuda.current_device())
        if case["op"] == "adapters":
            for t, rows in ((TABLE_A, s["a"]), (TABLE_B, s["b"])):
                srv.CreateTable(t, psa.TableInfo(row_capacity=rows.shape[1], max_rows=rows.shape[0]))
                srv.load_rows(t, 0, rows.cpu().numpy())
            first = [sum(s["ranks"][:i]) for i in range(len(s["ranks"]))]
            s["set"] = srv.create_adapters(TABLE_A, TABLE_B, list(zip(first, s["ranks"], s["scales"])))
        elif case["op"] == "bias":
            srv.CreateTable(TABLE_BIAS, psa.TableInfo(row_capacity=case["heads"], max_rows=case["buckets"]))
            srv.load_rows(TABLE_BIAS, 0, s["w"].cpu().numpy())
            s["bias"] = srv.position_bias(TABLE_BIAS, 0, case["buckets"], case["distance"], case["both"])
    if case["op"] == "adapters":
        s["out"] = torch.zeros_like(s["base"])
        if case["backward"]:   # what the forward pass left: x A^T, and x or its checkpoint
            if own:
                s["shrunk"] = s["set"].forward(s["x"], s["begin"], s["which"], out=torch.zeros_like(s["dy"]))[1]
                if case["checkpoint"]:
                    s["x"] = srv.checkpoint_store(s["x"])
            else:
                s["shrunk"] = _masked(s, s["x"].float() @ s["a"].t())
                if case["checkpoint"]:
                    s["x"] = _stored(s["x"])
    return s


# ---- the plain forms -----------------------------------------------------------------------------


def _masked(s, v):
    """v [tokens, all rank rows] times its scale where the token's adapter has the row, else zero."""
    token = torch.arange(v.shape[0], device=v.device, dtype=torch.int32)
    n = torch.bucketize(token, s["begin"], right=True) - 1
    inside = n < s["which"].numel()
    adapter = torch.where(inside, s["which"][n.clamp(max=s["which"].numel() - 1)], -1)
    owner = torch.repeat_interleave(torch.arange(len(s["ranks"]), device=v.device),
                                    torch.tensor(s["ranks"], device=v.device))
    scale = torch.tensor(s["scales"], device=v.device, dtype=v.dtype)[owner]
    return torch.where(adapter[:, None] == owner[None, :], v * scale, 0)


def _padded(s, out, value):
    """value in the rows that belong to a request; the rows behind the last stay."""
    token = torch.arange(out.shape[0], device=out.device)
    return torch.where((token < s["begin"][-1])[:, None], value.to(out.dtype), out)


def _grouped(x):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)


def _stored(x):
    """int8 values and their exponents, 32 values a group."""
    v = _grouped(x.float())
    fraction, power = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = (power - torch.where(fraction <= 127 / 128, 7, 6)).clamp(-126, 122)
    return (v * _power(-e)).round().to(torch.int8), e.to(torch.int8), x.shape[1], x.dtype


def _power(e):
    """2^e, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _loaded(stored, dtype=None):
    q, e, cols, kind = stored
    return (q * _power(e)).flatten(1)[:, :cols].to(dtype or kind)


def _borders(half, distance):
    """Distances at which the buckets behind the first half // 2 start: the least n with
    (n / exact)^m >= (distance / exact)^j, in whole numbers."""
    exact = half // 2
    m = half - exact

    def least(j):
        lo, hi = exact, distance
        at = distance ** j * exact ** (m - j)
        while lo < hi:
            n = (lo + hi) // 2
            lo, hi = (lo, n) if n ** m >= at else (n + 1, hi)
        return lo

    return [least(j) for j in range(1, m)]


def _buckets(case, relative):
    half = case["buckets"] // 2 if case["both"] else case["buckets"]
    n = relative.abs() if case["both"] else (-relative).clamp(min=0)
    borders = torch.tensor(_borders(half, case["distance"]) or [1 << 62], device=n.device)
    far = half // 2 + torch.bucketize(n, borders, right=True)
    b = torch.where(n < half // 2, n, far)
    return b + half * (relative > 0) if case["both"] else b


def _relative(case, begin, device):
    """The distances k - q that occur, from the least."""
    return torch.arange(-(case["q"] - 1) - begin, case["k"] - begin, device=device)


def run(s):
    case = s["case"]
    if case["op"] == "adapters":
        return _run_adapters(s, case)
    if case["op"] == "checkpoint":
        if own:
            kept = s["server"].checkpoint_store(s["x"])
            return kept.load()
        return _loaded(_stored(s["x"]))
    if case["backward"]:
        if own:
            return s["bias"].backward(s["d"], s["begin"], s["gain"])
        d = s["d"].float().sum(0)
        by_distance = _diagonals(d, case["q"], case["k"])
        bucket = _buckets(case, _relative(case, s["begin"], d.device))
        hot = (bucket[:, None] == torch.arange(case["buckets"], device=d.device)).double()
        return (s["gain"] * (by_distance.double() @ hot)).t().float().contiguous()
    if own:
        return s["bias"].forward(case["q"], case["k"], s["begin"], DTYPES[case["dtype"]])
    bucket = _buckets(case, _relative(case, s["begin"], s["w"].device))
    at = torch.arange(case["k"], device=bucket.device) - torch.arange(case["q"], device=bucket.device)[:, None]
    return s["w"].t()[:, bucket][:, at + case["q"] - 1].to(DTYPES[case["dtype"]])


def _run_adapters(s, case):
    if not case["backward"]:
        if own:
            return s["set"].forward(s["x"], s["begin"], s["which"], base=s["base"], out=s["out"])[0]
        v = _masked(s, s["x"].float() @ s["a"].t())
        return _padded(s, s["out"], s["base"].float() + v @ s["b"])
    if own:
        grad_a, grad_b = s["set"].backward(s["x"], s["dy"], s["shrunk"], s["begin"], s["which"], base=s["base"],
                                           out=s["out"], scale=s["gain"])
        return {"dx": s["out"], "grad_a": grad_a, "grad_b": grad_b}
    dy = s["dy"].float()
    x = _loaded(s["x"], torch.float32) if case["checkpoint"] else s["x"].float()
    u = _masked(s, dy @ s["b"].t())
    return {"dx": _padded(s, s["out"], s["base"].float() + u @ s["a"]),
            "grad_a": s["gain"] * (u.t() @ x), "grad_b": s["gain"] * (s["shrunk"].t() @ dy)}


def _diagonals(d, q, k):
    """Sums of d [heads, q, k] over each k - q, from -(q - 1): rows padded to q + k, read one short."""
    wide = torch.nn.functional.pad(d.flip(1), (0, q))
    return wide.flatten(1)[:, : q * (q + k - 1)].reshape(d.shape[0], q, q + k - 1).sum(1)


# ---- the work of one pass, and its exact result ------------------------------------------------------


def work(case):
    if case["op"] == "checkpoint":
        n, groups = case["rows"] * case["cols"], case["rows"] * (-(-case["cols"] // 32))
        return {"bytes": 2 * n * SIZES[case["dtype"]] + 2 * (n + groups), "flops": 4 * n}
    if case["op"] == "bias":
        n = case["batch"] * case["heads"] * case["q"] * case["k"]
        return {"bytes": n * SIZES[case["dtype"]] + 4 * case["buckets"] * case["heads"],
                "flops": n if case["backward"] else 0}
    T, d_in, d_out, es = case["tokens"], case["d_in"], case["d_out"], SIZES[case["dtype"]]
    ranks = _adapter_ranks(case)
    rank = sum(ranks) / len(ranks)
    rows = sum(ranks[: min(case["adapters"], case["requests"])])
    if case["backward"]:
        x = d_in * (33 / 32 if case["checkpoint"] else es)
        return {"bytes": T * (d_out * es + x + 2 * d_in * es + 4 * rank) + 4 * rows * (d_in + d_out)
                + 4 * sum(ranks) * (d_in + d_out), "flops": 4 * T * rank * (d_in + d_out)}
    return {"bytes": T * (d_in + 2 * d_out) * es + 4 * rows * (d_in + d_out), "flops": 2 * T * rank * (d_in + d_out)}


def exact(case, seed):
    if case["op"] == "checkpoint":
        return _exact_checkpoint(_activation(case, seed))
    if case["op"] == "bias":
        return _exact_bias(case, _bias_inputs(case, seed))
    s = _adapter_inputs(case, seed)
    T = case["tokens"] + case["pad"]
    out = torch.zeros(T, case["d_in"] if case["backward"] else case["d_out"], dtype=torch.float64, device="cuda")
    cuts, which = s["begin"].tolist(), s["which"].tolist()
    first = [sum(s["ranks"][:i]) for i in range(len(s["ranks"]) + 1)]
    x, base = s["x"].double(), s["base"].double()
    if case["checkpoint"]:
        kept = _exact_checkpoint(s["x"])
    grad_a, grad_b = (torch.zeros(first[-1], w, dtype=torch.float64, device="cuda") for w in (case["d_in"], case["d_out"]))
    for n, i in enumerate(which):
        at = slice(cuts[n], cuts[n + 1])
        if i < 0:
            out[at] = base[at]
            continue
        rows = slice(first[i], first[i + 1])
        a, b = s["a"][rows].double(), s["b"][rows].double() * s["scales"][i]
        v = x[at] @ a.t()
        if not case["backward"]:
            out[at] = base[at] + v @ b
            continue
        dy = s["dy"][at].double()
        u = dy @ b.t()
        out[at] = base[at] + u @ a
        grad_a[rows] += s["gain"] * (u.t() @ (kept if case["checkpoint"] else x)[at])
        grad_b[rows] += s["gain"] * s["scales"][i] * (v.t() @ dy)
    return {"dx": out, "grad_a": grad_a, "grad_b": grad_b} if case["backward"] else out


def _exact_checkpoint(x):
    """q 2^e of each 32 values: e the least integer whose 127 steps reach the largest of them."""
    v = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    top = v.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 127)), -126.0)

    def two_to(e):   # exactly, which a power function need not be
        return ((e.long() + 1023) << 52).view(torch.float64)

    e = torch.where(127 * two_to(e - 1) >= top, e - 1, e)
    e = torch.where(127 * two_to(e) < top, e + 1, e).clamp(-126, 122)
    return (torch.round(v * two_to(-e)) * two_to(e)).flatten(1)[:, : x.shape[1]]


def _exact_bias(case, s):
    q, k = case["q"], case["k"]
    half = case["buckets"] // 2 if case["both"] else case["buckets"]
    near, m = half // 2, half - half // 2

    def bucket(r):
        n = abs(r) if case["both"] else max(0, -r)
        b = n
        if n >= near:
            b = near + sum(n ** m * near ** j >= case["distance"] ** j * near ** m for j in range(1, m))
        return b + (half if case["both"] and r > 0 else 0)

    memo = {r: bucket(max(-case["distance"], min(case["distance"], r)))
            for r in range(-(q - 1) - s["begin"], k - s["begin"])}
    if not case["backward"]:
        table = torch.tensor([memo[r] for r in sorted(memo)], device="cuda")
        at = torch.arange(k, device="cuda")[None, :] - torch.arange(q, device="cuda")[:, None] + (q - 1)
        return s["w"].double().t()[:, table[at]] if case["heads"] * q * k <= 1 << 28 else None
    out = torch.zeros(case["buckets"], case["heads"], dtype=torch.float64, device="cuda")
    d = s["d"].double().sum(0)
    for r in sorted(memo):
        out[memo[r]] += torch.diagonal(d, offset=r + s["begin"], dim1=1, dim2=2).sum(1)
    return s["gain"] * out
