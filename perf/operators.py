"""Cases, plain forms and user calls of the token-path operators.

The operators carry tokens into and through a TAGI transformer: every value is a
Gaussian, held as a mean and a variance.

* ``lookup``      scaled embedding lookup: z = s w[id], mean and variance
* ``sums``        its gradient: the sums of the deltas over the tokens of each row
* ``update``      the same sums put straight into the capped update of the table
* ``norm``        residual addition and root-mean-square norm
* ``norm_back``   its backward pass, with the deltas of the scale parameters
* ``norm8``       residual addition and norm with the output in 8 bits
* ``linear8``     mean and variance of a linear layer from 8-bit operands with a
                  scale for each token and each channel

``own`` chooses between the plain forms (elementary torch operations) and the
calls of ``triton_tagi``. ``exact`` states the same results in 64 bits.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-6


def _kernels():
    """The package's kernel functions (reached only where ``own`` is true)."""
    if "triton_tagi" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "triton-tagi_b200"))
    from triton_tagi import kernels

    return kernels


# -- cases ----------------------------------------------------------------------


def _lookup(tokens, vocab, dim, scale, pad, ids):
    return {"op": "lookup", "tokens": tokens, "vocab": vocab, "dim": dim, "scale": scale,
            "pad": pad, "ids": ids, "skew": True}


def _grad(op, tokens, vocab, dim, scale, pad, ids, skew):
    return {"op": op, "tokens": tokens, "vocab": vocab, "dim": dim, "scale": scale, "pad": pad,
            "ids": ids, "skew": skew}


def _rows(op, rows, dim):
    return {"op": op, "rows": rows, "dim": dim}


def _linear(rows, inner, outer, bias):
    return {"op": "linear8", "rows": rows, "inner": inner, "outer": outer, "bias": bias}


def listed():
    return [
        # the next token of eight sequences that are being continued
        {"name": "lookup, 8 tokens", **_lookup(8, 32000, 512, 1.0, -1, "int32")},
        # a training batch of 32 sequences of 512, rows scaled by sqrt(dim)
        {"name": "lookup, 16384 tokens", **_lookup(16384, 32000, 512, math.sqrt(512), 0, "int64")},
        # the token-reversal task: 64 rows share 16384 tokens, ids as a Sequential passes them
        {"name": "sums, 64 rows", **_grad("sums", 16384, 64, 512, 1.0, -1, "float32", False)},
        # a text batch: few ids take most of the tokens, padded, odd sizes
        {"name": "update, text batch", **_grad("update", 65001, 50021, 770, math.sqrt(770), 0,
                                               "int64", True)},
        # one new token each of four sequences
        {"name": "norm, 4 rows", **_rows("norm", 4, 512)},
        # wide activations of a training batch
        {"name": "norm, 8192 x 4096", **_rows("norm", 8192, 4096)},
        # the token-reversal transformer's activations: 32 x 512 tokens of 512
        {"name": "norm_back, 16384 x 512", **_rows("norm_back", 16384, 512)},
        # the same activations on their way into an 8-bit layer
        {"name": "norm8, 16384 x 512", **_rows("norm8", 16384, 512)},
        # a ragged prompt of an odd width
        {"name": "norm8, 777 x 1001", **_rows("norm8", 777, 1001)},
        # three tokens through a down projection: latency, and the weights' bytes
        {"name": "linear8, 3 rows", **_linear(3, 2048, 512, True)},
        # the token-reversal transformer's up projection over a whole batch
        {"name": "linear8, 16384 x 512 x 2048", **_linear(16384, 512, 2048, True)},
        # the largest of the linear sweep
        {"name": "linear8, 8192 x 4096 x 4096", **_linear(8192, 4096, 4096, True)},
    ]


def _span(rng, low, high):
    """A whole number, even over the logarithm of the range."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "sums", "update", "norm", "norm_back", "norm8", "linear8",
                     "linear8"])
    if op == "lookup":
        return _lookup(_span(rng, 1, 30000), _span(rng, 64, 60000), _span(rng, 32, 1100),
                       rng.choice([1.0, 22.5]), rng.choice([-1, 0]),
                       rng.choice(["int32", "int64", "float32"]))
    if op in ("sums", "update"):
        return _grad(op, _span(rng, 16, 60000), _span(rng, 64, 50000), _span(rng, 32, 770),
                     rng.choice([1.0, 22.5]), rng.choice([-1, 0]),
                     rng.choice(["int32", "int64", "float32"]), rng.random() < 0.6)
    if op in ("norm", "norm_back", "norm8"):
        dim = _span(rng, 64, 5000)
        rows = _span(rng, 1, 16000)
        return _rows(op, min(rows, 8192 * 4096 // dim), dim)
    rows, inner, outer = _span(rng, 1, 8192), _span(rng, 64, 4096), _span(rng, 64, 4096)
    return _linear(rows, inner, outer, rng.random() < 0.7)


# -- inputs ---------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _uniform(g, low, high, *shape):
    return torch.rand(*shape, device="cuda", generator=g) * (high - low) + low


def _ids(case, g):
    """Token ids: even over the vocabulary, or (skewed) with probability falling as
    1/id, as words of a text do; a padded batch ends its sequences early."""
    n, V = case["tokens"], case["vocab"]
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    if case["skew"]:
        ids = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
    else:
        ids = (u * V).long().clamp_(0, V - 1)
    if case["pad"] >= 0:
        place = torch.arange(n, device="cuda") % 512
        ends = torch.randint(256, 513, ((n + 511) // 512,), device="cuda", generator=g)
        ids = torch.where(place < ends.repeat_interleave(512)[:n], ids, case["pad"])
    return ids.to(getattr(torch, case["ids"]))


def _codes_of(p, top):
    """Codes of the rows of a 64-bit tensor, and the largest magnitude of each row
    (rounded to 32 bits, as a scale is stored)."""
    most = p.abs().amax(-1, keepdim=True).float()
    return torch.round(p * top / most.double()), most


def _placed(codes, dtype):
    """Codes in 8 bits whose rows start on 16-byte boundaries."""
    rows, width = codes.shape
    buf = torch.zeros(rows, (width + 15) // 16 * 16, device="cuda", dtype=dtype)
    buf[:, :width] = codes.to(dtype)
    return buf[:, :width]


def _operand(first, second, third):
    q_m, a = _codes_of(first, 127.0)
    q_2, b = _codes_of(second, 255.0)
    q_S, c = _codes_of(third, 255.0)
    scales = torch.cat([a / 127.0, b / 255.0, c / 255.0], dim=1).t().contiguous()
    return (_placed(q_m, torch.int8), _placed(q_2, torch.uint8), _placed(q_S, torch.uint8), scales)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("lookup", "sums", "update"):
        V, D, n = case["vocab"], case["dim"], case["tokens"]
        s["ids"] = _ids(case, g)
        if op != "sums":
            s["mw"] = _normal(g, V, D) * 0.25
            s["Sw"] = _uniform(g, 0.5, 1.5, V, D) * 0.0625
        if op != "lookup":
            # deltas that come back through a scaled lookup are smaller by its scale
            s["dm"] = _normal(g, n, D) * (1e-2 / case["scale"])
            s["dS"] = -_uniform(g, 0.0, 1e-2 / case["scale"] ** 2, n, D)
    elif op in ("norm", "norm_back", "norm8"):
        R, D = case["rows"], case["dim"]
        s["mw"] = 1.0 + 0.1 * _normal(g, D)
        s["Sw"] = _uniform(g, 0.5, 1.5, D) / D
        if op == "norm_back":
            s["h"] = _normal(g, R, D) * 1.4
            h_S = _uniform(g, 2e-4, 2e-2, R, D)
            mean = (s["h"].double().square() + h_S.double()).mean(-1)
            s["inv"] = (mean + EPS).rsqrt().float()
            s["dm"] = _normal(g, R, D) * 1e-2
            s["dS"] = -_uniform(g, 0.0, 1e-2, R, D)
            s["rm"] = _normal(g, R, D) * 1e-2
            s["rS"] = -_uniform(g, 0.0, 1e-2, R, D)
        else:
            s["ma"], s["mr"] = _normal(g, R, D), _normal(g, R, D)
            s["Sa"], s["Sr"] = _uniform(g, 1e-4, 1e-2, R, D), _uniform(g, 1e-4, 1e-2, R, D)
    else:
        M, K, N = case["rows"], case["inner"], case["outer"]
        m, S = _normal(g, M, K).double(), _uniform(g, 1e-4, 1e-2, M, K).double()
        s["x"] = _operand(m, m * m, S)
        m = _normal(g, N, K).double() / math.sqrt(K)
        S = _uniform(g, 0.5, 1.5, N, K).double() / K
        s["w"] = _operand(m, m * m + S, S)
        if case["bias"]:
            s["mb"], s["Sb"] = _normal(g, N) * 0.1, _uniform(g, 0.5, 1.5, N) * 1e-3
        else:
            s["mb"] = s["Sb"] = None
    return s


# -- the operators ----------------------------------------------------------------


def _run_lookup(s):
    c = s["case"]
    if own:
        return _kernels().embedding_lookup(s["ids"], s["mw"], s["Sw"], scale=c["scale"],
                                           padding_idx=c["pad"])
    ids = s["ids"].long()
    keep = (ids != c["pad"]).float().unsqueeze(-1)
    return s["mw"][ids] * (keep * c["scale"]), s["Sw"][ids] * (keep * (c["scale"] * c["scale"]))


def _plain_sums(s, vocab):
    """Sums over the tokens of each row: long ones, so in 64 bits."""
    c = s["case"]
    ids = s["ids"].long()
    keep = (ids != c["pad"]).double().unsqueeze(-1)
    sums = []
    sums.append(torch.zeros(vocab, c["dim"], device="cuda", dtype=torch.float64).index_add_(
        0, ids, s["dm"].double() * keep) * c["scale"])
    sums.append(torch.zeros(vocab, c["dim"], device="cuda", dtype=torch.float64).index_add_(
        0, ids, s["dS"].double() * keep) * (c["scale"] * c["scale"]))
    return sums


def _run_sums(s):
    c = s["case"]
    if own:
        return _kernels().embedding_grad(s["ids"], s["dm"], s["dS"], c["vocab"],
                                         scale=c["scale"], padding_idx=c["pad"])
    g_m, g_S = _plain_sums(s, c["vocab"])
    return g_m.float(), g_S.float()


CAP = 3.0


def _run_update(s):
    c = s["case"]
    mw, Sw = s["mw"], s["Sw"]
    if own:
        _kernels().embedding_update(s["ids"], s["dm"], s["dS"], mw, Sw, CAP, scale=c["scale"],
                                    padding_idx=c["pad"])
        return mw, Sw
    g_m, g_S = _plain_sums(s, c["vocab"])
    d_m, d_S = g_m * Sw, g_S * Sw * Sw
    bound = Sw.double().clamp_min(1e-10).sqrt() / CAP
    mw.copy_(mw + torch.minimum(torch.maximum(d_m, -bound), bound))
    S = Sw + torch.minimum(torch.maximum(d_S, -bound), bound)
    Sw.copy_(torch.where(S <= 0, 1e-5, S))
    return mw, Sw


def _run_norm(s):
    if own:
        h_m, h_S, mz, Sz, inv = _kernels().add_rmsnorm(s["ma"], s["Sa"], s["mr"], s["Sr"],
                                                       s["mw"], s["Sw"], eps=EPS)
        return h_m, h_S, mz, Sz, inv
    w, Sw = s["mw"], s["Sw"]
    h_m, h_S = s["ma"] + s["mr"], s["Sa"] + s["Sr"]
    inv = 1.0 / torch.sqrt((h_m * h_m + h_S).mean(-1, keepdim=True) + EPS)
    mz = inv * h_m * w
    Sz = inv * inv * (h_S * (w * w + Sw) + Sw * h_m * h_m)
    return h_m, h_S, mz, Sz, inv.squeeze(-1)


def _run_norm_back(s):
    if own:
        return _kernels().add_rmsnorm_backward(s["dm"], s["dS"], s["h"], s["inv"], s["mw"],
                                               s["Sw"], s["rm"], s["rS"])
    inv = s["inv"].unsqueeze(-1)
    j = inv * s["mw"]
    x = inv * s["h"]
    g_m = (x * s["dm"]).double().sum(0)
    g_S = (x * x * s["dS"]).double().sum(0)
    return (s["rm"] + j * s["dm"], s["rS"] + j * j * s["dS"], (g_m * s["Sw"]).float(),
            (g_S * s["Sw"] * s["Sw"]).float())


def _run_norm8(s):
    if own:
        h_m, h_S, q = _kernels().add_rmsnorm_int8(s["ma"], s["Sa"], s["mr"], s["Sr"], s["mw"],
                                                  s["Sw"], eps=EPS)
        return (h_m, h_S, *q.values())
    w, Sw = s["mw"].double(), s["Sw"].double()
    h_m, h_S = s["ma"] + s["mr"], s["Sa"] + s["Sr"]
    inv = 1.0 / torch.sqrt((h_m * h_m + h_S).mean(-1, keepdim=True) + EPS)
    # a code is a whole number: values next to the middle between two are told apart in 64 bits
    p = h_m.double() * w
    t = h_S.double() * (w * w + Sw) + Sw * h_m.double().square()
    p_max, t_max = p.abs().amax(-1, keepdim=True).float(), t.amax(-1, keepdim=True).float()
    r = p / p_max.double()
    a = inv * p_max
    return (h_m, h_S, torch.round(127.0 * r).float() * (a / 127.0),
            torch.round(255.0 * r * r).float() * (a * a / 255.0),
            torch.round(255.0 * t / t_max.double()).float() * (inv * inv * t_max / 255.0))


def _run_linear8(s):
    if own:
        k = _kernels()
        return k.int8_moments_matmul(k.Int8Moments(*s["x"]), k.Int8Moments(*s["w"]), s["mb"],
                                     s["Sb"])
    xm, x2, xS = (t.float() for t in s["x"][:3])
    wm, w2, wS = (t.float() for t in s["w"][:3])
    a, b = s["x"][3].unsqueeze(-1), s["w"][3].unsqueeze(1)
    mz = (xm @ wm.t()) * (a[0] * b[0])
    Sz = (x2 @ wS.t()) * (a[1] * b[2]) + (xS @ w2.t()) * (a[2] * b[1])
    if s["mb"] is not None:
        mz, Sz = mz + s["mb"], Sz + s["Sb"]
    return mz, Sz


_RUN = {"lookup": _run_lookup, "sums": _run_sums, "update": _run_update, "norm": _run_norm,
        "norm_back": _run_norm_back, "norm8": _run_norm8, "linear8": _run_linear8}


def run(state):
    return _RUN[state["case"]["op"]](state)


# -- work -------------------------------------------------------------------------


def _touched(case):
    """Expected number of different ids among the tokens."""
    n, V = case["tokens"], case["vocab"]
    if case["skew"]:
        v = np.arange(V, dtype=np.float64)
        p = np.log((v + 2.0) / (v + 1.0)) / math.log(V + 1.0)
    else:
        p = np.full(V, 1.0 / V)
    share = 0.75 if case["pad"] >= 0 else 1.0
    return float(np.sum(-np.expm1(n * share * np.log1p(-p))))


def work(case):
    op = case["op"]
    if op in ("lookup", "sums", "update"):
        n, V, D = case["tokens"], case["vocab"], case["dim"]
        id_bytes = n * (8 if case["ids"] == "int64" else 4)
        real = n * (0.75 if case["pad"] >= 0 else 1.0)
        if op == "lookup":
            return {"bytes": id_bytes + 8 * D * (_touched(case) + n), "flops": 2 * n * D}
        if op == "sums":
            return {"bytes": id_bytes + 8 * D * (real + V), "flops": 2 * real * D}
        rows = _touched(case)
        return {"bytes": id_bytes + 8 * D * (real + 2 * rows), "flops": 2 * real * D + 12 * rows * D}
    if op in ("norm", "norm_back", "norm8"):
        R, D = case["rows"], case["dim"]
        per = {"norm": 32, "norm_back": 28, "norm8": 27}[op]
        return {"bytes": per * R * D + 16 * R + 16 * D, "flops": 14 * R * D}
    M, K, N = case["rows"], case["inner"], case["outer"]
    return {"bytes": 3 * M * K + 3 * N * K + 8 * M * N + 12 * (M + N), "flops": 6 * M * N * K}


# -- the definitions in 64 bits -----------------------------------------------------


def _segment_sums(ids, values, vocab):
    """Sums of the rows of `values` that share an id, by differences of running sums
    over the rows in the order of their ids."""
    order = torch.argsort(ids, stable=True)
    running = torch.cumsum(values.double()[order], 0)
    running = torch.cat([torch.zeros_like(running[:1]), running])
    edges = torch.searchsorted(ids[order], torch.arange(vocab + 1, device=ids.device))
    return running[edges[1:]] - running[edges[:-1]]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "ids"}
    if op in ("lookup", "sums", "update"):
        ids, pad, f = s["ids"].long(), case["pad"], case["scale"]
        if op == "lookup":
            d["mw"] = d["mw"] * f
            d["Sw"] = d["Sw"] * f ** 2
            if pad >= 0:
                d["mw"][pad] = 0.0
                d["Sw"][pad] = 0.0
            return d["mw"].index_select(0, ids), d["Sw"].index_select(0, ids)
        V = case["vocab"]
        g_m, g_S = _segment_sums(ids, d["dm"], V) * f, _segment_sums(ids, d["dS"], V) * f ** 2
        if pad >= 0:
            g_m[pad] = 0.0
            g_S[pad] = 0.0
        if op == "sums":
            return g_m, g_S
        S = d["Sw"]
        bound = S.clamp_min(1e-10) ** 0.5 / CAP
        step_m, step_S = S * g_m, S ** 2 * g_S
        m = d["mw"] + step_m.sign() * torch.minimum(step_m.abs(), bound)
        S = S + step_S.sign() * torch.minimum(step_S.abs(), bound)
        return m, torch.where(S > 0, S, 1e-5)
    if op == "norm_back":
        x = d["h"] * d["inv"][:, None]
        j = torch.outer(d["inv"], d["mw"])
        return (d["rm"] + j * d["dm"], d["rS"] + j ** 2 * d["dS"],
                d["Sw"] * torch.einsum("rd,rd->d", x, d["dm"]),
                d["Sw"] ** 2 * torch.einsum("rd,rd->d", x ** 2, d["dS"]))
    if op in ("norm", "norm8"):
        # the stream is held in 32 bits, and the norm reads it as it is held
        h = (s["ma"] + s["mr"]).double()
        v = (s["Sa"] + s["Sr"]).double()
        inv = ((h ** 2 + v).sum(-1) / case["dim"] + EPS) ** -0.5
        if op == "norm":
            h_m, h_S = d["ma"] + d["mr"], d["Sa"] + d["Sr"]
            w2 = d["mw"] ** 2
            return (h_m, h_S, h * d["mw"] * inv[:, None],
                    (v * w2 + v * d["Sw"] + h ** 2 * d["Sw"]) * (inv ** 2)[:, None], inv)
        p = d["mw"] * h
        t = d["Sw"] * (h ** 2 + v) + v * d["mw"] ** 2
        p_max = p.abs().max(-1).values.float().double()[:, None]
        t_max = t.max(-1).values.float().double()[:, None]
        top = inv[:, None] * p_max
        return (d["ma"] + d["mr"], d["Sa"] + d["Sr"], torch.round(p * 127.0 / p_max) * top / 127.0,
                torch.round((p / p_max) ** 2 * 255.0) * top ** 2 / 255.0,
                torch.round(t * 255.0 / t_max) * (inv ** 2)[:, None] * t_max / 255.0)
    x = [t.double() * k.double()[:, None] for t, k in zip(s["x"][:3], s["x"][3])]
    w = [t.double() * k.double()[:, None] for t, k in zip(s["w"][:3], s["w"][3])]
    mz = torch.einsum("mk,nk->mn", x[0], w[0])
    Sz = torch.einsum("mk,nk->mn", x[1], w[2]) + torch.einsum("mk,nk->mn", x[2], w[1])
    if case["bias"]:
        mz, Sz = mz + d["mb"][None], Sz + d["Sb"][None]
    return mz, Sz
