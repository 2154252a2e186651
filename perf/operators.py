"""The row operators of `nerfslam.rows` as measurable cases: embedding lookup with scaling, its gradient by sorted tokens, layer
norm and its backward pass.  `run` computes a case in elementary torch operations (`own` false) or through the framework (`own`
true) on the same inputs; `exact` states the same outputs in 64 bits."""
import math
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

EPS = 1e-5
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one new token of a decoder: nothing but latency
        dict(name="lookup_one_token", op="lookup", tokens=1, rows=32000, dim=1024, type="bf16", ids="int64", spread="zipf", pad=False, scale=32.0),
        # a latent per keyframe (512 slots: the tracker's buffer), one lookup per sample of a training step's 2^18 samples of 4096 rays
        dict(name="lookup_sample_views", op="lookup", tokens=262144, rows=512, dim=32, type="f16", ids="int32", spread="runs", pad=False, scale=1.0),
        # a long batch of text tokens, padded, over a vocabulary
        dict(name="lookup_vocabulary", op="lookup", tokens=65536, rows=50000, dim=2048, type="bf16", ids="int64", spread="zipf", pad=True, scale=45.25),
        # a ragged batch over a small table in single precision
        dict(name="lookup_grad_ragged", op="lookup_grad", tokens=3001, rows=1013, dim=771, type="f32", grad="f32", ids="int64", spread="even", pad=True, scale=0.5),
        # gradient of the keyframes' latents: few rows, 2^18 samples, every row hit hundreds of times
        dict(name="lookup_grad_sample_views", op="lookup_grad", tokens=262144, rows=512, dim=32, type="f16", grad="f32", ids="int32", spread="runs", pad=False, scale=1.0),
        # gradient of a vocabulary's table: a few rows hit by a tenth of the tokens, most by one or none
        dict(name="lookup_grad_vocabulary", op="lookup_grad", tokens=16384, rows=50000, dim=1024, type="bf16", grad="bf16", ids="int64", spread="zipf", pad=True, scale=32.0),
        # one new token's features
        dict(name="norm_one_row", op="norm", rows=1, dim=1024, type="bf16", weights="bf16"),
        # channels-last activations of 48 edges at 60 x 80 with 128 channels: the update operator's hidden state
        dict(name="norm_edge_maps", op="norm", rows=230400, dim=128, type="f16", weights="f32"),
        # a long batch of tokens
        dict(name="norm_tokens", op="norm", rows=16384, dim=4096, type="bf16", weights="bf16"),
        # the backward pass of the three kinds: ragged, channels-last maps, tokens
        dict(name="norm_grad_ragged", op="norm_grad", rows=257, dim=771, type="f32", weights="f32"),
        dict(name="norm_grad_edge_maps", op="norm_grad", rows=230400, dim=128, type="f16", weights="f32"),
        dict(name="norm_grad_tokens", op="norm_grad", rows=16384, dim=4096, type="bf16", weights="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("lookup", "lookup_grad", "norm", "norm_grad"))
    kind = rng.choice(("f16", "bf16", "f32"))
    dim = _log(rng, 1, 4096)
    if rng.random() < 0.5 and dim > 16:
        dim = dim // 8 * 8
    if op in ("norm", "norm_grad"):
        room = (1 << 26) // (2 if kind == "f32" else 1)
        return dict(op=op, rows=_log(rng, 1, min(230400, room // dim)), dim=dim, type=kind, weights=rng.choice((kind, "f32")))
    rows = _log(rng, 1, min(100000, (1 << 25) // dim))
    tokens = _log(rng, 1, min(262144, (1 << 25) // dim))
    case = dict(op=op, tokens=tokens, rows=rows, dim=dim, type=kind, ids=rng.choice(("int32", "int64")),
                spread=rng.choice(("zipf", "even", "runs")), pad=rng.random() < 0.5, scale=rng.choice((1.0, 0.5, 32.0, 45.25)))
    if op == "lookup_grad":
        case["grad"] = rng.choice((kind, "f32"))
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _ids(case, g, dev):
    n, rows = case["tokens"], case["rows"]
    if case["spread"] == "zipf":       # frequency ~ 1 / rank, ranks scattered over the table
        u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
        rank = (torch.exp(u * math.log(rows + 1.0)).floor().long() - 1).clamp_(0, rows - 1)
        ids = torch.randperm(rows, generator=g, device=dev)[rank]
    elif case["spread"] == "runs":     # the samples of a ray follow each other: 64 equal ids in a row
        m = (n + 63) // 64
        ids = torch.randint(0, rows, (m,), generator=g, device=dev).repeat_interleave(64)[:n]
    else:
        ids = torch.randint(0, rows, (n,), generator=g, device=dev)
    if case["pad"]:                    # padded places carry -1
        ids = torch.where(torch.rand(n, generator=g, device=dev) < 0.03, torch.full_like(ids, -1), ids)
    return ids.to(torch.int32 if case["ids"] == "int32" else torch.int64).contiguous()


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    t = _TYPES[case["type"]]
    if case["op"] == "lookup":
        return dict(ids=_ids(case, g, dev), table=(0.02 * normal(case["rows"], case["dim"])).to(t))
    if case["op"] == "lookup_grad":
        return dict(ids=_ids(case, g, dev), dout=normal(case["tokens"], case["dim"]).to(t))
    n, d, w = case["rows"], case["dim"], _TYPES[case["weights"]]
    x = (1.5 * normal(n, d) + 0.5 * normal(d) + 0.3).to(t)
    st = dict(x=x, weight=(1.0 + 0.1 * normal(d)).to(w), bias=(0.1 * normal(d)).to(w))
    if case["op"] == "norm_grad":
        st["dout"] = normal(n, d).to(t)
        x64 = x.double()               # the statistics that the forward pass left
        mean = x64.mean(1)
        var = (x64 - mean[:, None]).square().mean(1)
        st["mean"], st["rstd"] = mean.float(), (1.0 / torch.sqrt(var + EPS)).float()
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = dict(case)
    if own:
        at = os.path.join(ROOT, "nerf-slam_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        from nerfslam import rows
        st["rows"] = rows
    return st


# ---------------------------------------------------------------------------------------------- one pass
def _framework(st):
    c, rows = st["case"], st["rows"]
    if c["op"] == "lookup":
        return rows.embedding(st["table"], st["ids"], scale=c["scale"])
    if c["op"] == "lookup_grad":
        return rows.embedding_backward(st["dout"], st["ids"], c["rows"], scale=c["scale"], dtype=_TYPES[c["grad"]])
    if c["op"] == "norm":
        return rows.layer_norm(st["x"], st["weight"], st["bias"], eps=EPS, stats=True)
    return rows.layer_norm_backward(st["dout"], st["x"], st["mean"], st["rstd"], st["weight"])


def _plain(st):
    c = st["case"]
    if c["op"] == "lookup":
        ids = st["ids"].long()
        live = (ids >= 0) & (ids < c["rows"])
        out = st["table"][torch.where(live, ids, 0)].float() * c["scale"]
        return torch.where(live[:, None], out, 0.0).to(st["table"].dtype)
    if c["op"] == "lookup_grad":
        ids = st["ids"].long()
        live = (ids >= 0) & (ids < c["rows"])
        acc = torch.zeros((c["rows"] + 1, c["dim"]), dtype=torch.float32, device=ids.device)
        acc.index_add_(0, torch.where(live, ids, c["rows"]), st["dout"].float())
        return (acc[:-1] * c["scale"]).to(_TYPES[c["grad"]])
    x = st["x"].float()
    w = st["weight"].float()
    if c["op"] == "norm":
        mean = x.mean(1)
        x = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((x * x).mean(1) + EPS)
        return (x * rstd[:, None] * w + st["bias"].float()).to(st["x"].dtype), mean, rstd
    dout, rstd = st["dout"].float(), st["rstd"][:, None]
    xhat = (x - st["mean"][:, None]) * rstd
    g = dout * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(st["x"].dtype), (dout * xhat).sum(0).to(st["weight"].dtype), dout.sum(0).to(st["weight"].dtype)


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- what it has to do
def _distinct(case):
    """expected number of table rows that a case's tokens name"""
    v = case["rows"]
    live = case["tokens"] * (0.97 if case["pad"] else 1.0)
    if case["spread"] == "zipf":
        r = np.arange(1, v + 1, dtype=np.float64)
        return float((1.0 - np.exp(-live * np.log1p(1.0 / r) / math.log(v + 1.0))).sum())
    draws = live / 64.0 if case["spread"] == "runs" else live
    return float(v * (1.0 - math.exp(-max(draws, 1.0) / v)))


def work(case):
    d, e = case["dim"], _SIZE[case["type"]]
    if case["op"] in ("lookup", "lookup_grad"):
        n, v = case["tokens"], case["rows"]
        idb = 4 if case["ids"] == "int32" else 8
        if case["op"] == "lookup":
            return dict(bytes=int(n * idb + n * d * e + min(_distinct(case), n) * d * e), flops=n * d)
        return dict(bytes=int(n * idb + n * d * e * (0.97 if case["pad"] else 1.0) + v * d * _SIZE[case["grad"]]), flops=n * d + v * d)
    n, w = case["rows"], _SIZE[case["weights"]]
    if case["op"] == "norm":
        return dict(bytes=2 * n * d * e + 2 * d * w + 8 * n, flops=8 * n * d)
    return dict(bytes=3 * n * d * e + 3 * d * w + 8 * n, flops=14 * n * d)


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "lookup":
        ids, n = st["ids"].long(), case["rows"]
        table = torch.cat([st["table"].double() * case["scale"], torch.zeros((1, case["dim"]), dtype=torch.float64, device=ids.device)])
        return table.index_select(0, torch.where((ids < 0) | (ids >= n), torch.full_like(ids, n), ids))
    if case["op"] == "lookup_grad":
        ids, n = st["ids"].long(), case["rows"]
        keep = torch.nonzero((ids >= 0) & (ids < n))[:, 0]
        out = torch.zeros((n, case["dim"]), dtype=torch.float64, device=ids.device)
        for part in keep.split(65536):
            out.index_put_((ids[part],), st["dout"][part].double(), accumulate=True)
        return out.mul_(case["scale"])
    x, w = st["x"].double(), st["weight"].double()
    d = case["dim"]
    if case["op"] == "norm":
        mean = x.sum(1) / d
        var = (x * x).sum(1) / d - mean * mean
        rstd = (var.clamp_min(0.0) + EPS) ** -0.5
        return torch.addcmul(st["bias"].double().expand_as(x), (x - mean[:, None]) * w, rstd[:, None].expand_as(x)), mean, rstd
    dout, mean, rstd = st["dout"].double(), st["mean"].double(), st["rstd"].double()
    n = (x - mean[:, None]).mul_(rstd[:, None])
    dw, db = torch.linalg.vecdot(dout, n, dim=0), dout.sum(0)
    g = dout.mul_(w)
    a, b = g.sum(1) / d, torch.linalg.vecdot(g, n, dim=1) / d
    return (g - a[:, None] - n * b[:, None]).mul_(rstd[:, None]), dw, db
