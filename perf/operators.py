"""The operators on unit codes whose speed this package answers for.

A *code* is the position of one active unit: a sampled hidden layer, a complementary-coded binary image or a sequence of
tokens is a few codes per sample instead of a row of zeros and ones.  ``op`` names the operator:

``lookup``     the support that coded samples give: the sum of the weight rows that a sample's codes name, scaled
``gradient``   its gradient with respect to the weights: for every weight row the scaled sum over the codes that name it
``sample``     one unit per hypercolumn drawn from the softmax of the support, with temperature, top-k, top-p and min-p, from
               given random numbers: the codes the next layer looks up, or the answer
``loss``       distillation: the divergence of a student's hypercolumns from a teacher of which only the top units are kept
``distill``    the same with its gradient with respect to the student's support

``rows`` samples; ``codes`` codes a sample naming ``n`` weight rows of ``m`` units; ``hc`` hypercolumns of ``mc`` units; ``k``
units that are kept of the teacher.  A code of -1 names nothing.
"""
import math
from types import SimpleNamespace

import numpy as np
import torch

own = False   # True: the package's operators; False: their plain form


def listed():
    return [
        # one complementary-coded binary image through the MNIST hidden layer (784 of 1568 inputs, 30 x 100 units): a serving call
        dict(name="lookup_image_f32", op="lookup", dtype="float32", index="int32", rows=1, codes=784, n=1568, m=3000, coding="pairs", scale=1.0),
        # token embeddings of a training batch
        dict(name="lookup_tokens_bf16", op="lookup", dtype="bfloat16", index="int64", rows=16384, codes=1, n=50000, m=1024, coding="words", scale=32.0),
        # the output layer on the sampled codes of 30 hypercolumns of 100 units, one batch of 128: latency is all there is
        dict(name="gradient_classes_f32", op="gradient", dtype="float32", index="int64", rows=128, codes=30, n=3000, m=10, coding="units", scale=1.0),
        # odd sizes, short samples among long ones, double precision
        dict(name="gradient_ragged_f64", op="gradient", dtype="float64", index="int32", rows=1501, codes=5, n=10007, m=333, coding="ragged", scale=0.5),
        # the gradient of an embedding table, a few words in a good part of the places
        dict(name="gradient_tokens_bf16", op="gradient", dtype="bfloat16", index="int64", rows=65536, codes=1, n=50000, m=1024, coding="words", scale=32.0),
        # the next token of one sequence
        dict(name="sample_one_f16", op="sample", dtype="float16", rows=1, hc=1, mc=32000, temperature=0.8, top_k=50, top_p=0.9, min_p=0.0, per_row=False, masked=0.0),
        # a hidden layer of 30 x 100 units made binary, a large batch
        dict(name="sample_hidden_f32", op="sample", dtype="float32", rows=4096, hc=30, mc=100, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, per_row=False, masked=0.0),
        # a serving batch in which every sequence has settings of its own and a part of the tokens is ruled out
        dict(name="sample_batch_bf16", op="sample", dtype="bfloat16", rows=256, hc=1, mc=128000, temperature=0.7, top_k=100, top_p=0.95, min_p=0.02, per_row=True, masked=0.1),
        # a classifier of ten classes held against a teacher's best three, in double precision: evaluation
        dict(name="loss_classes_f64", op="loss", dtype="float64", index="int64", rows=8192, hc=1, mc=10, k=3, temperature=2.0, weighted=False),
        # validation of a student with a large output, odd in size
        dict(name="loss_tokens_f16", op="loss", dtype="float16", index="int32", rows=512, hc=1, mc=50001, k=32, temperature=1.0, weighted=True),
        # the wide hidden layer (100 x 300 units) learning from a larger one
        dict(name="distill_hidden_f32", op="distill", dtype="float32", index="int32", rows=1024, hc=100, mc=300, k=8, temperature=2.0, weighted=False),
        # a training batch of sequences, part of it padding
        dict(name="distill_tokens_bf16", op="distill", dtype="bfloat16", index="int64", rows=4096, hc=1, mc=32000, k=64, temperature=1.0, weighted=True),
    ]


def draw(rng):
    """One more case of the same ranges: every operator and type, sizes spread over their logarithm, most of them odd."""
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    while True:
        op = rng.choice(["lookup", "gradient", "sample", "loss", "distill"])
        c = dict(op=op, dtype=rng.choice(["float32", "float32", "bfloat16", "float16", "float64"]))
        width = {"float32": 4, "float64": 8}.get(c["dtype"], 2)
        if op in ("lookup", "gradient"):
            coding = rng.choice(["pairs", "words", "units", "ragged"])
            codes = 1 if coding == "words" else size(2, 1000)
            c.update(index=rng.choice(["int32", "int64"]), rows=size(1, 65536), codes=codes, coding=coding, m=size(1, 4096))
            c["n"] = 2 * codes if coding == "pairs" else 100 * codes if coding == "units" else size(2, 100000)
            if rng.random() < 0.5:
                c["m"] = (c["m"] + 7) // 8 * 8
            c["scale"] = rng.choice([1.0, 0.5, round(math.sqrt(c["m"]), 3)])
            entries = c["rows"] * codes
            if entries <= 1 << 18 and entries * c["m"] * width <= 128 << 20 and c["n"] * c["m"] * width <= 128 << 20:
                return c
            continue
        one = rng.random() < 0.5   # one wide group a row, or hypercolumns
        c.update(rows=size(1, 4096), hc=1 if one else size(1, 100), mc=size(500, 128000) if one else size(2, 500))
        if op == "sample":
            c.update(temperature=round(rng.uniform(0.3, 2.0), 2), top_k=rng.choice([0, 0, size(1, 200)]), top_p=rng.choice([1.0, 0.9, 0.5]),
                     min_p=rng.choice([0.0, 0.0, 0.05]), per_row=rng.random() < 0.3, masked=rng.choice([0.0, 0.0, 0.3]))
        else:
            c.update(index=rng.choice(["int32", "int64"]), k=min(c["mc"], size(1, 128)), temperature=rng.choice([1.0, 2.0, 4.0]), weighted=rng.random() < 0.5)
        if c["rows"] * c["hc"] * c["mc"] <= 32 << 20:
            return c


def _codes(c, gen):
    rows, k, n = c["rows"], c["codes"], c["n"]
    u = torch.rand((rows, k), generator=gen, device="cuda", dtype=torch.float64)
    if c["coding"] == "pairs":       # complementary-coded pixels: one input of each pair is active
        codes = 2 * torch.arange(k, device="cuda") + (u < 0.2)
    elif c["coding"] == "units":     # one unit of each hypercolumn
        per = n // k
        codes = per * torch.arange(k, device="cuda") + (u * per).long()
    elif c["coding"] == "words":     # word frequencies fall with their rank; words stand in any order in the table
        order = torch.randperm(n, generator=gen, device="cuda")
        codes = order[(torch.exp(u * math.log(n + 1)) - 1).long().clamp_(0, n - 1)]
    else:                            # samples of different lengths, filled up with -1
        length = torch.randint(0, k + 1, (rows, 1), generator=gen, device="cuda")
        codes = torch.where(torch.arange(k, device="cuda") < length, (u * n).long(), -1)
    return codes.to(getattr(torch, c["index"]))


def _support(c, gen, spread=3.0):
    return torch.randn((c["rows"], c["hc"] * c["mc"]), generator=gen, device="cuda").mul_(spread)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = getattr(torch, c["dtype"])
    s = SimpleNamespace(**{k: v for k, v in c.items() if k not in ("name", "dtype", "index", "coding", "codes", "masked")})
    if c["op"] == "lookup":
        s.weights = torch.randn((c["n"], c["m"]), generator=gen, device="cuda").to(dt)
        s.codes = _codes(c, gen)
        return s
    if c["op"] == "gradient":
        s.grad = torch.randn((c["rows"], c["m"]), generator=gen, device="cuda").to(dt)
        s.codes = _codes(c, gen)
        return s
    x = _support(c, gen)
    if c["op"] == "sample":
        if c["masked"]:
            x.masked_fill_(torch.rand(x.shape, generator=gen, device="cuda") < c["masked"], -math.inf)
        s.random = torch.rand((c["rows"], c["hc"]), generator=gen, device="cuda")
        if c["per_row"]:   # every row between greedy and twice as wild
            f = torch.rand((4, c["rows"]), generator=gen, device="cuda")
            s.temperature = torch.where(f[0] < 0.1, 0.0, 2 * c["temperature"] * f[0])
            s.top_k = (2 * c["top_k"] * f[1]).int()
            s.top_p = 1 - 2 * (1 - c["top_p"]) * f[2]
            s.min_p = 2 * c["min_p"] * f[3]
        s.support = x.to(dt)
        return s
    # the teacher's support is the student's with something added, and of it the best k units are kept
    t, u = (x + torch.randn(x.shape, generator=gen, device="cuda")).view(c["rows"], c["hc"], c["mc"]).topk(c["k"], dim=2)
    s.support, s.teacher_support, s.teacher_units = x.to(dt), t.to(dt), u.to(getattr(torch, c["index"]))
    s.weight = None
    if c["weighted"]:   # a tenth of the samples is padding
        s.weight = (torch.rand(c["rows"], generator=gen, device="cuda") >= 0.1).to(_wide(dt))
    return s


def _wide(dt):
    return torch.float64 if dt == torch.float64 else torch.float32


def _named(codes, n):
    return (codes >= 0) & (codes < n)


def _plain_lookup(s):
    codes, wide = s.codes.long(), _wide(s.weights.dtype)
    named = _named(codes, s.n)
    rows = s.weights[torch.where(named, codes, 0)].to(wide) * named[:, :, None].to(wide)
    return (rows.sum(1) * s.scale).to(s.weights.dtype)


def _plain_gradient(s):
    codes, wide = s.codes.long().reshape(-1), _wide(s.grad.dtype)
    named = _named(codes, s.n)
    rows = s.grad.to(wide)[torch.arange(codes.numel(), device=codes.device) // s.codes.shape[1]] * named[:, None].to(wide)
    total = torch.zeros((s.n, s.m), dtype=wide, device=codes.device).index_add_(0, torch.where(named, codes, 0), rows)
    return (total * s.scale).to(s.grad.dtype)


def _column(v, s, dtype):
    """A setting as a column with a value for every hypercolumn of every sample."""
    v = torch.as_tensor(v, device="cuda").to(dtype)
    return (v.view(-1, 1).expand(s.rows, s.hc) if v.dim() else v.expand(s.rows, s.hc)).reshape(-1, 1)


def _plain_sample(s):
    # in 64 bits: a number next to the border of two units has to fall on the right side of it
    x = s.support.double().view(-1, s.mc)
    x = torch.where(torch.isnan(x), -math.inf, x)
    t, k = _column(s.temperature, s, torch.float64), _column(s.top_k, s, torch.int64)
    p, low = _column(s.top_p, s, torch.float64), _column(s.min_p, s, torch.float64)
    best = x.max(1, keepdim=True).values
    w = torch.exp((x - best) / torch.where(t > 0, t, 1.0))
    w = torch.where(x == best, 1.0, w)
    w = torch.where(x == -math.inf, 0.0, w)
    k = torch.where(t > 0, torch.where(k > 0, k, s.mc), 1)
    order = x.sort(dim=1, descending=True, stable=True).indices
    rank = torch.arange(s.mc, device="cuda")
    ws = w.gather(1, order) * (rank < k)
    c = ws.cumsum(1)
    before = torch.cat((torch.zeros_like(c[:, :1]), c[:, :-1]), 1)
    keep = (rank < k) & ((before < p * c[:, -1:]) | (p >= 1) | (rank == 0)) & (ws >= low)
    w = w * torch.zeros_like(keep).scatter_(1, order, keep)
    c = w.cumsum(1)
    drawn = (c <= s.random.double().view(-1, 1) * c[:, -1:]).sum(1)
    last = torch.where(w > 0, rank, -1).max(1).values
    codes = torch.where(best[:, 0] > -math.inf, torch.minimum(drawn, last) + s.mc * torch.arange(s.hc, device="cuda").repeat(s.rows), -1)
    return codes.view(s.rows, s.hc)


def _plain_distill(s, gradient):
    wide = _wide(s.support.dtype)
    x = s.support.to(wide).view(s.rows, s.hc, s.mc) / s.temperature
    t = s.teacher_support.to(wide) / s.temperature
    units = s.teacher_units.long()
    x = x - x.max(2, keepdim=True).values
    e = torch.exp(x)
    total = e.sum(2, keepdim=True)
    t = t - t.max(2, keepdim=True).values
    p = torch.exp(t)
    mass = p.sum(2, keepdim=True)
    p = p / mass
    log_q = x.gather(2, units) - torch.log(total)
    weight = (torch.ones((), dtype=wide, device="cuda") if s.weight is None else s.weight)[..., None]
    loss = (p * (t - torch.log(mass) - log_q)).sum(2) * s.temperature ** 2 * weight
    if not gradient:
        return loss
    g = (e / total).scatter_add_(2, units, -p) * (s.temperature * weight[..., None])
    return {"loss": loss, "gradient": g.view(s.rows, -1).to(s.support.dtype)}


def run(state):
    s = state
    if own:
        from streambrain_b200 import kernels_device as k
        if s.op == "lookup":
            return k.lookup(s.weights, s.codes, scale=s.scale)
        if s.op == "gradient":
            return k.lookup_gradient(s.grad, s.codes, s.n, scale=s.scale)
        if s.op == "sample":
            return k.sample_minicolumns(s.support, s.hc, s.mc, s.random, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)
        if s.op == "loss":
            return k.distill_loss(s.support, s.hc, s.mc, s.teacher_units, s.teacher_support, temperature=s.temperature, weight=s.weight)
        loss, gradient = k.distill_gradient(s.support, s.hc, s.mc, s.teacher_units, s.teacher_support, temperature=s.temperature, weight=s.weight)
        return {"loss": loss, "gradient": gradient}
    if s.op == "lookup":
        return _plain_lookup(s)
    if s.op == "gradient":
        return _plain_gradient(s)
    if s.op == "sample":
        return _plain_sample(s)
    return _plain_distill(s, s.op == "distill")


def work(case):
    c = case
    e = {"float32": 4, "float64": 8}.get(c["dtype"], 2)
    if c["op"] in ("lookup", "gradient"):
        entries, i, m = c["rows"] * c["codes"], 8 if c["index"] == "int64" else 4, c["m"]
        if c["op"] == "gradient":
            return {"bytes": float(c["rows"] * m * e + entries * i + c["n"] * m * e), "flops": float(entries * m)}
        if c["coding"] == "words":   # the rows that some code names
            p = np.diff(np.log(np.arange(1, c["n"] + 2))) / math.log(c["n"] + 1)
        else:
            p = np.full(c["n"], (0.5 if c["coding"] == "ragged" else 1.0) / c["n"])
        touched = float(np.sum(-np.expm1(entries * np.log1p(-p)))) if c["n"] > 1 else 1.0
        if c["coding"] in ("pairs", "units") and c["rows"] == 1:
            touched = c["codes"]
        return {"bytes": float(touched * m * e + entries * i + c["rows"] * m * e), "flops": float(entries * m)}
    units = c["rows"] * c["hc"] * c["mc"]
    if c["op"] == "sample":
        return {"bytes": float(units * e + c["rows"] * c["hc"] * 12), "flops": float(4 * units)}
    kept = c["rows"] * c["hc"] * c["k"] * (e + (8 if c["index"] == "int64" else 4))
    return {"bytes": float(units * e * (2 if c["op"] == "distill" else 1) + kept + c["rows"] * c["hc"] * max(e, 4)), "flops": float((6 if c["op"] == "distill" else 4) * units)}


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "sample":
        return None   # whole numbers
    if s.op == "lookup":
        total = torch.zeros((s.rows, s.m), dtype=torch.float64, device="cuda")
        padded = torch.cat((s.weights.double(), torch.zeros((1, s.m), dtype=torch.float64, device="cuda")))   # what no code names is row n
        for j in range(s.codes.shape[1]):
            code = s.codes[:, j].long()
            total += padded[torch.where(code < 0, s.n, code)]
        return total * s.scale
    if s.op == "gradient":
        # runs of equal codes in sorted order, each the difference of two running sums
        code, order = s.codes.long().reshape(-1).sort(stable=True)
        end = torch.searchsorted(code, torch.arange(-1, s.n, device="cuda"), right=True)
        out = torch.empty((s.n, s.m), dtype=torch.float64, device="cuda")
        for lo in range(0, s.m, 256):
            part = s.grad[:, lo:lo + 256].double()[order // s.codes.shape[1]]
            run_ = torch.cat((torch.zeros_like(part[:1]), part.cumsum(0)))
            out[:, lo:lo + 256] = (run_[end[1:]] - run_[end[:-1]]) * s.scale
        return out
    x = s.support.double().view(s.rows, s.hc, s.mc) / s.temperature
    log_q = torch.log_softmax(x, 2)
    log_p = torch.log_softmax(s.teacher_support.double() / s.temperature, 2)
    weight = 1.0 if s.weight is None else s.weight.double()[:, None]
    units = s.teacher_units.long()
    loss = (log_p.exp() * (log_p - torch.gather(log_q, 2, units))).sum(2) * weight * s.temperature ** 2
    if s.op == "loss":
        return loss
    p = torch.zeros_like(x).scatter_(2, units, log_p.exp())
    g = (log_q.exp() - p) * s.temperature * (weight if s.weight is None else weight[:, :, None])
    return {"loss": loss, "gradient": g.reshape(s.rows, -1)}
