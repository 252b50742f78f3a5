"""Timed cases of the sequence model operators: ``rms_norm`` (with the residual's addition and the
8-bit output), ``causal_conv``, ``selective_scan`` and ``random.sample``.

With ``own`` false, ``run`` computes each operator in its plain form: elementary torch operations in
32 bits (64 for float64 inputs and for the cumulative probabilities of the sampler), rounded once at
the end.  With ``own`` true it makes the framework's calls: the operators are recorded once as a step
(``record``), and each pass submits that step, as a decoding loop does.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float16": torch.float16, "float32": torch.float32, "float64": torch.float64}
_DEVICE = "cuda"


# ---- cases ------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of four requests: a norm whose cost is its launch
        {"name": "norm token", "op": "norm", "rows": 4, "n": 2048, "dtype": "float16", "residual": True, "bits": 0, "group": 0},
        # a prompt's activations on their way into an 8-bit projection, one scale for 128 columns
        {"name": "norm prompt 8 bits", "op": "norm", "rows": 8192, "n": 4096, "dtype": "float16", "residual": True, "bits": 8, "group": 128},
        # rows whose length no vector width divides, in the framework's own 32 bits
        {"name": "norm odd", "op": "norm", "rows": 1531, "n": 5003, "dtype": "float32", "residual": True, "bits": 0, "group": 0},
        # four prompts of different lengths in one padded batch, carried state in and out
        {"name": "conv prompt", "op": "conv", "b": 4, "t": 4096, "d": 4096, "k": 4, "dtype": "float16", "ragged": True},
        # one token of each of 96 requests
        {"name": "conv token", "op": "conv", "b": 96, "t": 1, "d": 4100, "k": 4, "dtype": "float32", "ragged": False},
        # one long prompt: the largest case
        {"name": "scan prompt", "op": "scan", "b": 1, "t": 8192, "d": 4096, "n": 16, "dtype": "float16", "gate": True, "ragged": False},
        # prompts of odd and different lengths, one of them empty, continuing earlier states
        {"name": "scan ragged", "op": "scan", "b": 5, "t": 1003, "d": 1537, "n": 16, "dtype": "float32", "gate": True, "ragged": True},
        # one token of each of 128 requests: the states are read and written
        {"name": "scan token", "op": "scan", "b": 128, "t": 1, "d": 4096, "n": 16, "dtype": "float16", "gate": True, "ragged": False},
        # the framework's default type, as its solvers use it
        {"name": "scan double", "op": "scan", "b": 2, "t": 1000, "d": 500, "n": 12, "dtype": "float64", "gate": False, "ragged": False},
        # the end of one request's decoding step
        {"name": "sample one", "op": "sample", "rows": 1, "v": 32768, "dtype": "float32", "top_k": 0, "top_p": 0.95, "min_p": 0.0, "temperature": 0.8},
        # the end of a large batch's step; 16-bit logits are full of ties
        {"name": "sample many", "op": "sample", "rows": 128, "v": 131072, "dtype": "float16", "top_k": 50, "top_p": 0.9, "min_p": 0.02, "temperature": 0.7},
        # an odd vocabulary, a wide nucleus
        {"name": "sample odd", "op": "sample", "rows": 37, "v": 50021, "dtype": "float32", "top_k": 0, "top_p": 0.98, "min_p": 0.0, "temperature": 1.3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan", "sample"])
    dtype = rng.choice(["float16", "float16", "float32", "float32", "float64"])
    if op == "norm":
        n = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(8192, (8192 * 4096 // n) // (2 if dtype == "float64" else 1)))
        bits = rng.choice([0, 8])
        return {"op": op, "rows": rows, "n": n, "dtype": dtype, "residual": rng.random() < 0.7, "bits": bits,
                "group": rng.choice([0, 32, 128, _log(rng, 16, n)]) if bits else 0}
    if op == "conv":
        b, d = _log(rng, 1, 128), _log(rng, 64, 8192)
        t = 1 if rng.random() < 0.3 else _log(rng, 1, max(2, min(8192, (1 << 25) // (b * d))))
        return {"op": op, "b": b, "t": t, "d": d, "k": rng.randint(2, 8), "dtype": dtype, "ragged": rng.random() < 0.5}
    if op == "scan":
        b, d, n = _log(rng, 1, 128), _log(rng, 64, 8192), rng.choice([rng.randint(1, 16), 16, _log(rng, 16, 64)])
        most = (1 << 25) if dtype == "float64" else (1 << 28)
        t = 1 if rng.random() < 0.3 else _log(rng, 1, max(2, min(8192, most // (b * d * n))))
        return {"op": op, "b": b, "t": t, "d": d, "n": n, "dtype": dtype, "gate": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    v = _log(rng, 1000, 262144)
    return {"op": op, "rows": _log(rng, 1, max(1, min(256, (1 << 23) // v))), "v": v, "dtype": dtype,
            "top_k": rng.choice([0, 0, 1, _log(rng, 2, 1000), _log(rng, 2, v)]),
            "top_p": rng.choice([1.0, rng.uniform(0.1, 0.5), rng.uniform(0.5, 1.0)]),
            "min_p": rng.choice([0.0, 0.0, rng.uniform(0.005, 0.3)]), "temperature": rng.uniform(0.4, 1.6)}


def _bytes_of(case):
    return {"float16": 2, "float32": 4, "float64": 8}[case["dtype"]]


def _acc_bytes(case):
    return 8 if case["dtype"] == "float64" else 4


def work(case):
    e, a, op = _bytes_of(case), _acc_bytes(case), case["op"]
    if op == "norm":
        size = case["rows"] * case["n"]
        groups = -(-case["n"] // (case["group"] or case["n"]))
        moved = size * e * ((3 if case["residual"] else 1) + (0 if case["bits"] else 1)) + case["n"] * e
        if case["bits"]:
            # the codes and their scales, and the values they stand for
            moved += size * (1 + 1 + a) + 2 * case["rows"] * groups * a
        return {"bytes": moved, "flops": 6 * size}
    if op == "conv":
        size = case["b"] * case["t"] * case["d"]
        state = case["b"] * (case["k"] - 1) * case["d"]
        return {"bytes": e * (2 * size + 2 * state + case["d"] * (case["k"] + 1)), "flops": size * (2 * case["k"] + 5)}
    if op == "scan":
        size = case["b"] * case["t"] * case["d"]
        state = case["b"] * case["d"] * case["n"]
        return {"bytes": e * (size * (4 if case["gate"] else 3) + 2 * case["b"] * case["t"] * case["n"])
                + a * (2 * state + case["d"] * (case["n"] + 2)), "flops": size * (7 * case["n"] + 12)}
    return {"bytes": case["rows"] * (case["v"] * e + 4 + 4 + a), "flops": 4 * case["rows"] * case["v"]}


# ---- inputs -------------------------------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    acc = torch.float64 if case["dtype"] == "float64" else torch.float32

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=_DEVICE, dtype=torch.float32) * scale).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0, dtype=acc):
        u = torch.rand(shape, generator=g, device=_DEVICE, dtype=torch.float64 if dtype == torch.float64 else torch.float32)
        return (u * (hi - lo) + lo).to(dtype)

    def lengths(b, t):
        if not case["ragged"]:
            return None
        got = torch.randint(0, t + 1, (b,), generator=g, device=_DEVICE, dtype=torch.int32)
        got[0] = t
        return got

    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        # a residual stream: most columns of order one, a few large ones
        columns = torch.where(uniform(n) > 0.99, 8.0, 1.0).to(acc)
        return {"x": normal(rows, n), "residual": (normal(rows, n, dtype=acc) * columns).to(dt) if case["residual"] else None,
                "weight": normal(n, scale=0.2, dtype=acc).add(1.0).to(dt)}
    if case["op"] == "conv":
        b, t, d, k = case["b"], case["t"], case["d"], case["k"]
        return {"x": normal(b, t, d), "weight": normal(d, k, scale=k ** -0.5), "bias": normal(d, scale=0.1),
                "state": normal(b, k - 1, d), "lengths": lengths(b, t)}
    if case["op"] == "scan":
        b, t, d, n = case["b"], case["t"], case["d"], case["n"]
        step = torch.exp(uniform(d, lo=math.log(1e-3), hi=math.log(0.1)))
        return {"x": normal(b, t, d), "delta": normal(b, t, d, scale=0.5),
                "A": -(torch.arange(1, n + 1, device=_DEVICE).to(acc) * torch.exp(normal(d, n, scale=0.1, dtype=acc))),
                "B": normal(b, t, n), "C": normal(b, t, n), "D": normal(d, scale=0.1, dtype=acc).add(1.0),
                "z": normal(b, t, d) if case["gate"] else None,
                "delta_bias": step + torch.log(-torch.expm1(-step)),
                "state": normal(b, d, n, dtype=acc), "lengths": lengths(b, t)}
    rows, v = case["rows"], case["v"]
    return {"logits": normal(rows, v, scale=2.5, dtype=torch.float32).add(normal(rows, 1, scale=3.0, dtype=torch.float32)).to(dt),
            "u": uniform(rows)}


def prepare(case, seed):
    inputs = _inputs(case, seed)
    state = {"case": case, "inputs": inputs}
    if own:
        # a program of the framework has its data in the framework's arrays, and records its step once
        import charmnumeric_b200 as cnp
        interface = _interface(cnp)
        torch.cuda.synchronize()
        arrays = {k: None if v is None else cnp.from_device(interface, v) for k, v in inputs.items()}
        interface.context.synchronize()
        # one stream for both libraries: torch's kernels that read an output run behind the operator that makes it, and
        # the next pass, which writes it again, behind them
        stream = next(v for v in arrays.values() if v is not None).device_view(interface).stream
        torch.cuda.set_stream(torch.cuda.ExternalStream(stream))
        state.update(interface=interface, step=cnp.record(lambda: _OWN[case["op"]](cnp, case, arrays)), out=None)
        state["inputs"] = None
    return state


_open = []


def _interface(cnp):
    if not _open:
        _open.append(cnp.CharmNumericInterface(device=0))
    return _open[0]


def run(state):
    if own:
        state["step"].run(state["interface"])
        if state["out"] is None:
            # torch's view of the step's result arrays: the same memory from pass to pass
            state["out"] = {k: torch.as_tensor(v.device_view(state["interface"]), device=_DEVICE)
                            for k, v in state["step"].results.items()}
        return state["out"]
    return _PLAIN[state["case"]["op"]](state["case"], state["inputs"])


# ---- the framework's calls ----------------------------------------------------------------------------

def _own_norm(cnp, case, a):
    if case["bits"]:
        q, scale, *h = cnp.rms_norm(a["x"], a["weight"], residual=a["residual"], eps=1e-5, bits=8, group=case["group"] or None)
        out = {"y": cnp.dequantize(q, scale), "scale": scale}
    elif case["residual"]:
        y, *h = cnp.rms_norm(a["x"], a["weight"], residual=a["residual"], eps=1e-5)
        out = {"y": y}
    else:
        h, out = [], {"y": cnp.rms_norm(a["x"], a["weight"], eps=1e-5)}
    if h:
        out["h"] = h[0]
    return out


def _own_conv(cnp, case, a):
    y, state = cnp.causal_conv(a["x"], a["weight"], a["bias"], state=a["state"], lengths=a["lengths"], activation="silu")
    return {"y": y, "state": state}


def _own_scan(cnp, case, a):
    y, state = cnp.selective_scan(a["x"], a["delta"], a["A"], a["B"], a["C"], D=a["D"], z=a["z"], delta_bias=a["delta_bias"],
                                  state=a["state"], lengths=a["lengths"])
    return {"y": y, "state": state}


def _own_sample(cnp, case, a):
    token, logp = cnp.random.sample(a["logits"], a["u"], temperature=case["temperature"], top_k=case["top_k"],
                                    top_p=case["top_p"], min_p=case["min_p"])
    return {"token": token, "logp": logp}


_OWN = {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan, "sample": _own_sample}


# ---- plain forms --------------------------------------------------------------------------------------

def _acc(x):
    return x if x.dtype == torch.float64 else x.float()


def _plain_norm(case, a):
    x = a["x"]
    h = _acc(x) if a["residual"] is None else _acc(x) + _acc(a["residual"])
    r = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    if case["bits"]:
        # the codes do not depend on r: it is in the scale
        rows, n = h.shape
        size = case["group"] or n
        groups = -(-n // size)
        v = h * _acc(a["weight"])
        v = torch.cat([v, v.new_zeros(rows, groups * size - n)], 1).reshape(rows, groups, size)
        most = v.abs().amax(2, keepdim=True)
        codes = torch.round(v * torch.where(most > 0, 127.0 / most, 0.0)).to(torch.int8)
        scale = most * r[:, :, None] / 127.0
        out = {"y": (codes.to(h.dtype) * scale).reshape(rows, groups * size)[:, :n].contiguous(), "scale": scale[:, :, 0].contiguous()}
    else:
        out = {"y": (h * r * _acc(a["weight"])).to(x.dtype)}
    if a["residual"] is not None:
        out["h"] = h.to(x.dtype)
    return out


def _live(lengths, b, t, device):
    if lengths is None:
        return None
    return torch.arange(t, device=device)[None, :] < lengths[:, None]


def _plain_conv(case, a):
    x = a["x"]
    b, t, d = x.shape
    k = case["k"]
    padded = torch.cat([a["state"], x], 1)
    windows = _acc(padded).unfold(1, k, 1)
    s = (windows * _acc(a["weight"])).sum(3) + _acc(a["bias"])
    y = s / (1.0 + torch.exp(-s))
    if a["lengths"] is None:
        return {"y": y.to(x.dtype), "state": padded[:, t:].contiguous()}
    y = torch.where(_live(a["lengths"], b, t, x.device)[:, :, None], y, 0.0)
    at = a["lengths"][:, None].long() + torch.arange(k - 1, device=x.device)[None, :]
    return {"y": y.to(x.dtype), "state": torch.gather(padded, 1, at[:, :, None].expand(b, k - 1, d))}


def _plain_scan(case, a):
    x = a["x"]
    b, t, d = x.shape
    dt = _acc(a["delta"]) + a["delta_bias"]
    dt = torch.clamp(dt, min=0.0) + torch.log1p(torch.exp(-dt.abs()))
    live = _live(a["lengths"], b, t, x.device)
    if live is not None:
        dt = torch.where(live[:, :, None], dt, 0.0)
    decay = torch.exp(dt[..., None] * a["A"])
    h = (dt * _acc(x))[..., None] * _acc(a["B"])[:, :, None, :]
    h[:, 0] += decay[:, 0] * a["state"]
    # h_t = decay_t h_(t-1) + h_t by doubling: after each turn an entry holds twice as many steps
    step = 1
    while step < t:
        h = torch.cat([h[:, :step], torch.addcmul(h[:, step:], decay[:, step:], h[:, :-step])], 1)
        decay = torch.cat([decay[:, :step], decay[:, step:] * decay[:, :-step]], 1)
        step *= 2
    del decay
    y = (h * _acc(a["C"])[:, :, None, :]).sum(3) + a["D"] * _acc(x)
    if a["z"] is not None:
        z = _acc(a["z"])
        y = y * (z / (1.0 + torch.exp(-z)))
    if live is not None:
        y = torch.where(live[:, :, None], y, 0.0)
    return {"y": y.to(x.dtype), "state": h[:, -1].contiguous()}


def _plain_sample(case, a):
    # 64 bits: the running sum over a vocabulary is compared with a border
    x = a["logits"].double()
    rows, v = x.shape
    most = x.amax(1, keepdim=True)
    p = torch.exp((x - most) / case["temperature"])
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    best = torch.gather(p, 1, order)
    kept = torch.ones_like(best, dtype=torch.bool)
    if 0 < case["top_k"] < v:
        kept = kept & (torch.arange(v, device=x.device) < case["top_k"])
    best = torch.where(kept, best, 0.0)
    if case["top_p"] < 1.0:
        before = torch.cumsum(best, 1) - best
        kept = kept & (before < case["top_p"] * best.sum(1, keepdim=True))
    kept = kept & (best >= case["min_p"])
    kept = torch.zeros_like(kept).scatter(1, order, kept)
    p = torch.where(kept, p, 0.0)
    total = p.sum(1, keepdim=True)
    token = (torch.cumsum(p, 1) <= a["u"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=v - 1)
    logp = torch.log(torch.gather(p, 1, token) / total)
    return {"token": token[:, 0].to(torch.int32), "logp": logp[:, 0].to(torch.float64 if case["dtype"] == "float64" else torch.float32)}


_PLAIN = {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan, "sample": _plain_sample}


# ---- the definition in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    a = {k: None if v is None else (v.double() if v.is_floating_point() else v) for k, v in _inputs(case, seed).items()}
    return _EXACT[case["op"]](case, a)


def _exact_norm(case, a):
    h = a["x"] if a["residual"] is None else a["x"] + a["residual"]
    mean = torch.einsum("ij,ij->i", h, h) / case["n"] + 1e-5
    if not case["bits"]:
        out = {"y": h * a["weight"] * torch.rsqrt(mean)[:, None]}
    else:
        # what the codes stand for has no value of its own apart from its rounding to 8 bits
        size = case["group"] or case["n"]
        scaled = (h * a["weight"]).abs()
        most = torch.stack([part.amax(1) for part in scaled.split(size, 1)], 1)
        out = {"y": None, "scale": most / 127.0 * torch.rsqrt(mean)[:, None]}
    if a["residual"] is not None:
        out["h"] = h
    return out


def _exact_conv(case, a):
    b, t, d, k = (case[key] for key in ("b", "t", "d", "k"))
    y = torch.zeros(b, t, d, dtype=torch.float64, device=_DEVICE)
    state = torch.zeros(b, k - 1, d, dtype=torch.float64, device=_DEVICE)
    ends = [t] * b if a["lengths"] is None else a["lengths"].tolist()
    for i, end in enumerate(ends):
        row = torch.cat([a["state"][i], a["x"][i, :end]])
        s = a["bias"].repeat(end, 1)
        for j in range(k):
            s += row[j:j + end] * a["weight"][:, j]
        y[i, :end] = s * torch.sigmoid(s)
        state[i] = row[end:]
    return {"y": y, "state": state}


def _exact_scan(case, a):
    b, t, d, n = (case[key] for key in ("b", "t", "d", "n"))
    h = a["state"].clone()
    y = torch.zeros(b, t, d, dtype=torch.float64, device=_DEVICE)
    for i in range(t):
        dt = torch.nn.functional.softplus(a["delta"][:, i] + a["delta_bias"], threshold=700.0)
        new = torch.exp(dt[:, :, None] * a["A"]) * h + torch.einsum("bd,bn->bdn", dt * a["x"][:, i], a["B"][:, i])
        out = torch.einsum("bdn,bn->bd", new, a["C"][:, i]) + a["D"] * a["x"][:, i]
        if a["z"] is not None:
            out = out * a["z"][:, i] * torch.sigmoid(a["z"][:, i])
        if a["lengths"] is None:
            h, y[:, i] = new, out
        else:
            on = i < a["lengths"]
            h = torch.where(on[:, None, None], new, h)
            y[:, i] = torch.where(on[:, None], out, 0.0)
    return {"y": y, "state": h}


def _exact_sample(case, a):
    logits, u = a["logits"].cpu().numpy(), a["u"].cpu().numpy()
    tokens, logps = [], []
    for x, draw_ in zip(logits, u):
        z = x / case["temperature"]
        z = z - z.max()
        keep = np.argsort(-z, kind="stable")
        if case["top_k"]:
            keep = keep[:case["top_k"]]
        mass = np.exp(z[keep])
        if case["top_p"] < 1.0:
            keep = keep[:1 + np.count_nonzero(np.cumsum(mass)[:-1] < case["top_p"] * mass.sum())]
        keep = np.sort(keep[np.exp(z[keep]) >= case["min_p"]])
        run_ = np.cumsum(np.exp(z[keep]))
        at = min(np.searchsorted(run_, draw_ * run_[-1], side="right"), len(keep) - 1)
        tokens.append(keep[at])
        logps.append(z[keep[at]] - np.log(run_[-1]))
    return {"token": np.array(tokens, dtype=np.int32), "logp": np.array(logps)}


_EXACT = {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan, "sample": _exact_sample}
