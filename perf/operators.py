"""The learned-code operators, as they are measured: embedding lookup, layer norm and counter-based dropout.

Each case is one pass of one operator in one direction.  Where ``own`` is false, ``run`` computes the operator from
elementary torch operations; where it is true, it calls ``torch_nerf.amd.ops`` the way a training loop or a server does.

The generator of the dropout: element e of the global tensor (e = first + flat index) takes 32 bits of the 64-bit word
mix(key + (e >> 1) * 0xD1342543DE82EF95), the low half for an even e and the high half for an odd one, where mix is the
splitmix64 finaliser (the stream behind ``ops.counter_uniform``); it is kept iff those bits, as an unsigned number, are
>= round(p * 2^32).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_GAMMA, _M1, _M2 = 0xD1342543DE82EF95, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
_ops = None


def _framework():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "torch-nerf_amd"))
        from torch_nerf.amd import ops
        _ops = ops
    return _ops


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # serving: the one new token of a stream
        {"name": "embed_one_token", "op": "embed", "way": "fwd", "n": 1, "rows": 32768, "dim": 4096, "dtype": "bf16",
         "ids": "zipf", "scale": 64.0, "pad": False},
        # a training batch of tokens over a large vocabulary
        {"name": "embed_tokens", "op": "embed", "way": "fwd", "n": 16384, "rows": 131072, "dim": 2048, "dtype": "bf16",
         "ids": "zipf", "scale": math.sqrt(2048.0), "pad": False},
        # its gradient: frequent tokens repeat thousands of times, the ends of padded sequences give none
        {"name": "embed_grad_tokens", "op": "embed", "way": "bwd", "n": 16384, "rows": 131072, "dim": 1024, "dtype": "bf16",
         "ids": "zipf", "scale": 32.0, "pad": True},
        # latent codes of 100 views, one per ray, handed to all 64 + 128 samples of 4096 rays: few rows, each hit often
        {"name": "embed_grad_codes", "op": "embed", "way": "bwd", "n": 786432, "rows": 100, "dim": 48, "dtype": "fp32",
         "ids": "rays", "scale": 1.0, "pad": False},
        # serving: one hidden state
        {"name": "norm_one_row", "op": "norm", "way": "fwd", "rows": 1, "dim": 4096, "dtype": "bf16", "weight": "bf16"},
        # the features of 4096 x 64 samples
        {"name": "norm_samples", "op": "norm", "way": "fwd", "rows": 262144, "dim": 256, "dtype": "fp32", "weight": "fp32"},
        # odd row length: no row but the first starts on a vector's boundary
        {"name": "norm_odd", "op": "norm", "way": "fwd", "rows": 5003, "dim": 1365, "dtype": "fp16", "weight": "fp16"},
        # the features of 4096 x (64 + 128) samples, backward: the weight's gradient sums 786432 rows
        {"name": "norm_grad_samples", "op": "norm", "way": "bwd", "rows": 786432, "dim": 256, "dtype": "fp32",
         "weight": "fp32"},
        # a training batch of hidden states with master weights in fp32
        {"name": "norm_grad_tokens", "op": "norm", "way": "bwd", "rows": 8192, "dim": 4096, "dtype": "bf16",
         "weight": "fp32"},
        # the features of one small batch of points
        {"name": "dropout_small", "op": "dropout", "way": "fwd", "rows": 512, "dim": 256, "dtype": "fp32", "p": 0.1,
         "first": 0, "add": False},
        # the features of 4096 x (64 + 128) samples
        {"name": "dropout_samples", "op": "dropout", "way": "fwd", "rows": 786432, "dim": 256, "dtype": "bf16", "p": 0.1,
         "first": 0, "add": False},
        # a shard of a batch that begins at an odd element, added to a residual stream of odd size
        {"name": "dropout_add_odd", "op": "dropout", "way": "fwd", "rows": 16383, "dim": 2047, "dtype": "bf16", "p": 0.25,
         "first": 33536001, "add": True},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op, way = rng.choice(["embed", "norm", "dropout"]), rng.choice(["fwd", "bwd"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "embed":
        dim, rows = _log(rng, 1, 4096), _log(rng, 1, 131072)
        n = min(_log(rng, 1, 786432), max(1, 2 ** 27 // dim))
        rows = min(rows, max(1, 2 ** 27 // dim))
        return {"op": op, "way": way, "n": n, "rows": rows, "dim": dim, "dtype": dtype,
                "ids": rng.choice(["zipf", "rays", "even", "same"]), "scale": rng.choice([1.0, round(math.sqrt(dim), 4)]),
                "pad": way == "bwd" and rng.random() < 0.5}
    dim = _log(rng, 1, 16384)
    rows = min(_log(rng, 1, 786432), max(1, 2 ** 27 // dim))
    if op == "norm":
        return {"op": op, "way": way, "rows": rows, "dim": dim, "dtype": dtype, "weight": rng.choice([dtype, "fp32"])}
    return {"op": op, "way": way, "rows": rows, "dim": dim, "dtype": dtype, "p": rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9]),
            "first": rng.choice([0, rng.randrange(2 ** 20), rng.randrange(2 ** 40)]), "add": way == "fwd" and rng.random() < 0.5}


# --------------------------------------------------------------------------- inputs
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _ids(case, g):
    """int64 rows of the table.  zipf: words of a text; rays: one view per ray, for all of the ray's samples; even: any row
    is as likely as any other; same: one image's code for the whole batch."""
    n, rows, kind = case["n"], case["rows"], case["ids"]
    if kind == "zipf":
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        rank = torch.exp(u * math.log(rows)).long().sub_(1).clamp_(0, rows - 1)
        return torch.randperm(rows, generator=g, device="cuda")[rank]
    if kind == "rays":
        rays = torch.randint(rows, ((n + 191) // 192,), generator=g, device="cuda")
        return rays.repeat_interleave(192)[:n].contiguous()
    if kind == "same":
        return torch.randint(rows, (1,), generator=g, device="cuda").repeat(n)
    return torch.randint(rows, (n,), generator=g, device="cuda")


def prepare(case, seed):
    g, t = _gen(seed), DTYPES[case["dtype"]]

    def normal(*shape, dtype=t):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": case}
    if case["op"] == "embed":
        s["ids"] = _ids(case, g)
        s["pad"] = -1
        if case["pad"]:          # the last eighth of the batch is padding: row 0 stands for "no token"
            s["ids"][case["n"] - case["n"] // 8:] = 0
            s["pad"] = 0
        if case["way"] == "fwd":
            s["table"] = normal(case["rows"], case["dim"])
        else:
            s["g"] = normal(case["n"], case["dim"])
    elif case["op"] == "norm":
        w = DTYPES[case["weight"]]
        m, c = case["rows"], case["dim"]
        # activations: channels of different size, with an offset of their own
        size = torch.rand(c, generator=g, device="cuda") + 0.5
        off = torch.randn(c, generator=g, device="cuda") * 0.5
        s["x"] = torch.randn(m, c, generator=g, device="cuda").mul_(size).add_(off).to(t)
        s["w"] = (1.0 + 0.1 * torch.randn(c, generator=g, device="cuda")).to(w)
        s["b"] = normal(c, dtype=w)
        if case["way"] == "bwd":
            s["g"] = normal(m, c)
            s["mean"], s["rstd"] = _moments(s["x"])     # what the forward pass kept
    else:
        s["x"] = normal(case["rows"], case["dim"])
        s["r"] = normal(case["rows"], case["dim"]) if case["add"] else None
        s["key"] = (int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) % 2 ** 64
    return s


# --------------------------------------------------------------------------- the plain forms
EPS = 1e-5


def _moments(x):
    x = x.float()
    mean = x.mean(1)
    d = x - mean[:, None]
    return mean, torch.rsqrt((d * d).mean(1) + EPS)


def _signed(v):
    return v - 2 ** 64 if v >= 2 ** 63 else v


def _right(x, k):
    return (x >> k) & ((1 << (64 - k)) - 1)


def _kept(case, key, shape):
    """Truth values of the elements that stay."""
    n = shape[0] * shape[1]
    pair = case["first"] >> 1
    word = torch.arange(pair, pair + n // 2 + 2, device="cuda") * _signed(_GAMMA) + _signed(key)
    word = (word ^ _right(word, 30)) * _signed(_M1)
    word = (word ^ _right(word, 27)) * _signed(_M2)
    word = word ^ _right(word, 31)
    bits = torch.stack([word & 0xFFFFFFFF, _right(word, 32)], 1).reshape(-1)[case["first"] & 1:][:n]
    return (bits >= round(case["p"] * 2 ** 32)).view(shape)


def _plain(s):
    case = s["case"]
    if case["op"] == "embed":
        if case["way"] == "fwd":
            return (s["table"][s["ids"]].float() * case["scale"]).to(s["table"].dtype)
        live = (s["ids"] != s["pad"]).double()[:, None]
        total = torch.zeros(case["rows"], case["dim"], device="cuda", dtype=torch.float64)
        total.index_add_(0, s["ids"], s["g"].double() * live)
        return (total * case["scale"]).to(s["g"].dtype)
    if case["op"] == "norm":
        x, w = s["x"].float(), s["w"].float()
        if case["way"] == "fwd":
            mean, rstd = _moments(s["x"])
            y = (x - mean[:, None]) * rstd[:, None] * w + s["b"].float()
            return [y.to(s["x"].dtype), mean, rstd]
        h = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = s["g"].float()
        gw, gb = (g * h).sum(0, dtype=torch.float64), g.sum(0, dtype=torch.float64)
        g = g * w
        gx = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * s["rstd"][:, None]
        return [gx.to(s["x"].dtype), gw.to(s["w"].dtype), gb.to(s["w"].dtype)]
    y = torch.where(_kept(case, s["key"], s["x"].shape), s["x"].float() * (1.0 / (1.0 - case["p"])), 0.0)
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["x"].dtype)


def _call(s):
    ops, case = _framework(), s["case"]
    if case["op"] == "embed":
        if case["way"] == "fwd":
            return ops.embedding(s["table"], s["ids"], scale=case["scale"])
        return ops.embedding_backward(s["g"], s["ids"], case["rows"], scale=case["scale"],
                                      padding_idx=s["pad"] if case["pad"] else None)
    if case["op"] == "norm":
        if case["way"] == "fwd":
            return list(ops.layernorm(s["x"], s["w"], s["b"], EPS, want_stats=True))
        return list(ops.layernorm_backward(s["g"], s["x"], s["w"], s["mean"], s["rstd"]))
    if case["way"] == "fwd":
        return ops.dropout(s["x"], case["p"], s["key"], first=case["first"], residual=s["r"])
    return ops.dropout_backward(s["x"], case["p"], s["key"], first=case["first"])


def run(state):
    return _call(state) if own else _plain(state)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "embed":
        n, rows, dim = case["n"], case["rows"], case["dim"]
        if case["way"] == "fwd":
            seen = 1 if case["ids"] == "same" else min((n + 191) // 192 if case["ids"] == "rays" else n, rows)
            return {"bytes": 8 * n + size * dim * (seen + n), "flops": n * dim}
        return {"bytes": 8 * n + size * dim * (n + rows), "flops": n * dim}
    cells = case["rows"] * case["dim"]
    if case["op"] == "norm":
        w = 4 if case["weight"] == "fp32" else 2
        if case["way"] == "fwd":
            return {"bytes": 2 * size * cells + 2 * w * case["dim"] + 8 * case["rows"], "flops": 7 * cells}
        return {"bytes": 3 * size * cells + 3 * w * case["dim"] + 8 * case["rows"], "flops": 14 * cells}
    return {"bytes": (3 if case["add"] else 2) * size * cells, "flops": (2 if case["add"] else 1) * cells}


# --------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        ids = s["ids"].cpu().numpy()
        if case["way"] == "fwd":
            return s["table"].double().index_select(0, s["ids"]).mul_(case["scale"])
        # the rows of the gradient in the order of their ids, summed run by run
        g = s["g"].double().cpu().numpy()
        if case["pad"]:
            g, ids = g[ids != 0], ids[ids != 0]
        out = np.zeros((case["rows"], case["dim"]))
        if len(ids):
            order = np.argsort(ids, kind="stable")
            which, start = np.unique(ids[order], return_index=True)
            out[which] = np.add.reduceat(g[order], start, axis=0) * case["scale"]
        return torch.from_numpy(out)
    if case["op"] == "norm":
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        inv = 1.0 / torch.sqrt(var + EPS)
        h = (x - mean) * inv
        if case["way"] == "fwd":
            return [h * w + b, mean[:, 0], inv[:, 0]]
        g = s["g"].double()
        gw, gb = torch.linalg.vecdot(g, h, dim=0), g.sum(0)
        # the Jacobian of the norm applied to g * w: project out the constant and h, divide by the deviation
        g = g * w
        a, c = g.mean(1, keepdim=True), torch.linalg.vecdot(g, h, dim=1)[:, None] / case["dim"]
        return [inv * (g - a - c * h), gw, gb]
    # the generator on the host, in unsigned 64-bit numbers
    n = case["rows"] * case["dim"]
    keep = np.empty(n, bool)
    limit = int(math.floor(case["p"] * 2.0 ** 32 + 0.5))
    step = 1 << 24
    for lo in range(0, n, step):
        e = np.arange(lo, min(n, lo + step), dtype=np.uint64) + np.uint64(case["first"])
        z = (e >> np.uint64(1)) * np.uint64(_GAMMA) + np.uint64(s["key"])
        z = (z ^ (z >> np.uint64(30))) * np.uint64(_M1)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(_M2)
        z ^= z >> np.uint64(31)
        z = np.where(e % np.uint64(2) == 1, z >> np.uint64(32), z & np.uint64(0xFFFFFFFF))
        keep[lo:lo + len(e)] = z >= np.uint64(limit)
    y = s["x"].double() / (1.0 - case["p"])
    y[~torch.from_numpy(keep).cuda().view(y.shape)] = 0.0
    return y if s["r"] is None else y + s["r"].double()
