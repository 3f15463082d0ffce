"""Operators on unit codes against plain 64-bit implementations on the CPU, and their refusals.

Tolerances count roundings.  With u half a step of the type sums are held in (2^-24, for float64 2^-53), a sum of m terms is off
by at most m u times the sum of their magnitudes, and the result is rounded once more, by half a step of its own type (float16
also by half of its smallest number, 2^-25)."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from streambrain_b200 import _lib  # noqa: E402
from streambrain_b200._lib import lib  # noqa: E402

gpu = pytest.mark.gpu
F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16
ALL = [F32, F64, F16, BF16]


def half_step(t):
    return torch.finfo(t).eps / 2


def wide_half_step(t):
    return half_step(F64 if t == F64 else F32)


def rounding(t, value):
    return half_step(t) * value.abs() + (2.0 ** -25 if t == F16 else 0)


def assert_close(got, want, bound):
    got, off = got.double().cpu(), None
    assert got.shape == want.shape
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(off <= bound)
    assert not bad.any(), "%d of %d values off, the worst by %g where %g is allowed" % (
        bad.sum(), bad.numel(), off[bad].max(), (bound.expand_as(off)[bad]).max())


def values(shape, t, seed, spread=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape) * spread).to(t)


# ---- plain implementations -------------------------------------------------

def plain_lookup(weights, codes, scale):
    """(result, sum of magnitudes) in 64 bits."""
    w = weights.double()
    n = w.shape[0]
    c = codes.long()
    named = ((c >= 0) & (c < n)).double()[..., None]
    rows = w[torch.where(named[..., 0] > 0, c, 0)] * named
    return rows.sum(1) * scale, rows.abs().sum(1) * abs(scale)


def plain_gradient(grad, codes, n, scale):
    """(result, sum of magnitudes, number of terms of the fullest row) in 64 bits."""
    g, c = grad.double(), codes.long()
    out = torch.zeros((n, g.shape[1]), dtype=F64)
    size, count = torch.zeros_like(out), np.zeros(n, dtype=int)
    for r in range(c.shape[0]):
        row, row_size = g[r], g[r].abs()
        for code in c[r].tolist():
            if 0 <= code < n:
                out[code] += row
                size[code] += row_size
                count[code] += 1
    return out * scale, size * abs(scale), int(count.max()) if n else 0


def plain_sample(x, h, mc, random, temperature, top_k, top_p, min_p):
    """Loops over hypercolumns; 64 bits."""
    rows = x.shape[0]
    x = x.double().numpy().reshape(rows, h, mc)
    pick = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))   # (numbers are rounded to float32)
    out = np.full((rows, h), -1, dtype=np.int64)
    for r in range(rows):
        t, k, p, low = pick(temperature, r), int(pick(top_k, r)), pick(top_p, r), min(pick(min_p, r), 1.0)
        for g in range(h):
            v = np.where(np.isnan(x[r, g]), -np.inf, x[r, g])
            best = v.max()
            if best == -np.inf:
                continue
            with np.errstate(over="ignore", invalid="ignore"):
                w = np.where(v == best, 1.0, np.exp((v - best) / (t if t > 0 else 1.0)))
            order = sorted(range(mc), key=lambda i: (-v[i], i))
            if not t > 0:
                k = 1
            if k > 0:
                order = order[:k]
            total, before, kept = math.fsum(w[order]), 0.0, []
            for i in order:
                if kept and p < 1 and not before < p * total:
                    break
                kept.append(i)
                before = math.fsum(w[kept])
            kept = [i for i in kept if w[i] >= low or v[i] == best]
            total, u = math.fsum(w[kept]), float(random[r, g])
            run, unit = [], None
            for i in sorted(kept):
                run.append(w[i])
                if w[i] > 0:
                    unit = i
                if math.fsum(run) > u * total:
                    break
            out[r, g] = g * mc + unit
    return torch.from_numpy(out)


def plain_distill(x, h, mc, units, teacher, temperature, weight):
    """(loss, gradient, bound of the loss, bound of the gradient) in 64 bits.

    A weight exp((x - max) / t) is off by a few u and 3 u for each unit of its exponent, a sum of n of them by n u more (a
    kernel's partial sums are shorter), and so is what is divided by it; the loss adds k terms of such factors."""
    t = x.dtype
    u = wide_half_step(t)
    rows, k = x.shape[0], units.shape[2]
    x64 = x.double().reshape(rows, h, mc)
    units, t64 = units.long(), teacher.double()
    loss = torch.zeros((rows, h), dtype=F64)
    grad = torch.zeros((rows, h, mc), dtype=F64)
    loss_off, grad_off = torch.zeros_like(loss), torch.zeros_like(grad)
    for r in range(rows):
        w = 1.0 if weight is None else float(weight[r])
        for g in range(h):
            there = [j for j in range(k) if 0 <= units[r, g, j] < mc]
            v = x64[r, g]
            if w == 0 or not there or v.max() == -math.inf or t64[r, g, there].max() == -math.inf:
                continue
            named = units[r, g, there]
            tv = t64[r, g, there]
            log_q, log_p = torch.log_softmax(v / temperature, 0), torch.log_softmax(tv / temperature, 0)
            p, q = log_p.exp(), log_q.exp()
            terms = torch.where(p > 0, p * (log_p - log_q[named]), torch.zeros_like(p))
            pp = torch.zeros(mc, dtype=F64).index_add_(0, named, p)
            loss[r, g] = w * temperature ** 2 * terms.sum()
            grad[r, g] = w * temperature * (q - pp)
            finite = v[torch.isfinite(v)]
            span = float(((finite.max() - finite.min()) / temperature).clamp(max=120)) if len(finite) else 0.0
            tf = tv[torch.isfinite(tv)]
            tspan = float(((tf.max() - tf.min()) / temperature).clamp(max=120)) if len(tf) else 0.0
            c = (6 * max(span, tspan) + mc + k + 40) * u
            scale = torch.where(p > 0, p * (log_p.abs() + log_q[named].abs() + 1), torch.zeros_like(p)).sum()
            loss_off[r, g] = abs(w) * temperature ** 2 * scale * c + 1e-37
            grad_off[r, g] = abs(w) * temperature * (q + pp) * c + (1e-37 if t != F64 else 1e-300)
    return loss, grad.reshape(rows, -1), loss_off, grad_off.reshape(rows, -1)


def codes_of(kind, rows, length, n, seed, dtype):
    rng = np.random.default_rng(seed)
    if kind == "any":
        c = rng.integers(0, n, (rows, length))
    elif kind == "absent":     # some outside on either side, some rows empty
        c = rng.integers(-n, 2 * n, (rows, length))
        c[:: 3] = -1
    elif kind == "same":
        c = np.full((rows, length), n - 1)
    else:                      # a few words nearly everywhere
        c = np.minimum((n + 1) ** rng.random((rows, length)) - 1, n - 1).astype(np.int64)
    return torch.from_numpy(c.astype(np.int64)).to(dtype)


def k():
    from streambrain_b200 import kernels_device
    return kernels_device


# ---- lookup and its gradient -----------------------------------------------

LOOKUPS = [  # rows, codes, N, M, kind of codes, scale
    (1, 1, 1, 1, "any", 1.0), (1, 784, 1568, 300, "any", 1.0), (1, 5000, 97, 10, "any", 0.5), (3, 2, 5, 7, "absent", -2.0),
    (33, 1, 1000, 129, "few", 32.0), (128, 30, 3000, 10, "any", 1.0), (65, 9, 40, 1030, "absent", 0.25), (7, 31, 64, 2, "same", 1.0),
    (300, 1, 17, 64, "any", 8.0), (20, 100, 200, 2056, "few", 1.0), (2, 3, 11, 4100, "any", 1.0),
]


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,length,n,m,kind,scale", LOOKUPS)
def test_lookup(rows, length, n, m, kind, scale, t):
    w = values((n, m), t, 1)
    for index in (torch.int32, torch.int64):
        c = codes_of(kind, rows, length, n, 2, index)
        want, size = plain_lookup(w, c, scale)
        got = k().lookup(w.cuda(), c.cuda(), scale)
        assert got.dtype == t
        assert_close(got, want, (length + 2) * wide_half_step(t) * size + rounding(t, want))


GRADIENTS = LOOKUPS + [  # long runs of equal codes, runs that end anywhere, few and many codes for the table
    (700, 1, 3, 20, "any", 1.0), (1000, 3, 5000, 33, "few", 1.0), (40, 300, 50, 16, "same", 1.0), (5000, 2, 300, 9, "few", 1.0),
    (9001, 1, 20011, 8, "few", 1.0), (6000, 3, 100, 6, "any", 1.0), (36000, 1, 300, 4, "few", 1.0), (900, 99, 70001, 3, "absent", 1.0),
    (140001, 1, 1000, 2, "any", 1.0), (133, 1000, 40, 3, "any", 1.0), (70000, 2, 300, 1, "same", 1.0), (3, 1, 70001, 3, "any", 1.0), (130, 130, 700, 40, "absent", 1.0), (20000, 1, 9, 5, "any", 1.0),
]


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,length,n,m,kind,scale", GRADIENTS)
def test_lookup_gradient(rows, length, n, m, kind, scale, t):
    g = values((rows, m), t, 3)
    c = codes_of(kind, rows, length, n, 4, torch.int64)
    want, size, most = plain_gradient(g, c, n, scale)
    bound = (most + 2) * wide_half_step(t) * size + rounding(t, want)
    got = k().lookup_gradient(g.cuda(), c.cuda(), n, scale)
    assert_close(got, want, bound)
    again = k().lookup_gradient(g.cuda(), c.int().cuda(), n, scale)
    assert torch.equal(got, again)
    # added to what is there: one more addition, and the rows that no code names keep their bits
    old = values((n, m), t, 5)
    out = old.cuda()
    assert k().lookup_gradient(g.cuda(), c.cuda(), n, scale, out=out, accumulate=True) is out
    both = want + old.double()
    assert_close(out, both, bound + 2 * wide_half_step(t) * (old.double().abs() + size) + rounding(t, both))
    named = torch.zeros(n, dtype=torch.bool)
    named[c[(c >= 0) & (c < n)].long()] = True
    assert torch.equal(out.cpu()[~named], old[~named])


def gradient_by_torch(grad, codes, n):
    """(result, sum of magnitudes, number of terms of the fullest row) in 64 bits, on the tensors' device."""
    c = codes.long().reshape(-1)
    row = torch.arange(c.numel(), device=c.device) // codes.shape[1]
    keep = (c >= 0) & (c < n)
    c, row = c[keep], row[keep]
    out = torch.zeros((n, grad.shape[1]), dtype=F64, device=grad.device)
    size = torch.zeros_like(out)
    for lo in range(0, c.numel(), 1 << 20):
        g = grad.double()[row[lo:lo + (1 << 20)]]
        out.index_add_(0, c[lo:lo + (1 << 20)], g)
        size.index_add_(0, c[lo:lo + (1 << 20)], g.abs())
    return out, size, int(torch.bincount(c, minlength=n).max())


@gpu
@pytest.mark.parametrize("t,m", [(F16, 8), (BF16, 16), (BF16, 32), (F32, 16), (F64, 8), (BF16, 3)])
def test_lookup_gradient_of_millions_of_codes(t, m):
    """The longest chunks, in the narrowest rows: four lanes to a chunk, 64 chunks to a block."""
    rows, length, n = 8192, 600, 90001
    g, c = values((rows, m), t, 71).cuda(), codes_of("few", rows, length, n, 72, torch.int32).cuda()
    want, size, most = gradient_by_torch(g, c, n)
    got = k().lookup_gradient(g, c, n)
    assert_close(got, want.cpu(), ((most + 2) * wide_half_step(t) * size + rounding(t, want)).cpu())


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("kind", ["any", "few", "same", "absent"])
def test_lookup_gradient_of_long_chunks(kind, t):
    """Chunks of 16 to 64 entries (elsewhere they are of 8): some ten thousand codes of wide rows."""
    rows, n, m = 20011, 3001, 2048
    g, c = values((rows, m), t, 73).cuda(), codes_of(kind, rows, 1, n, 74, torch.int64).cuda()
    want, size, most = gradient_by_torch(g, c, n)
    got = k().lookup_gradient(g, c, n)
    assert_close(got, want.cpu(), ((most + 2) * wide_half_step(t) * size + rounding(t, want)).cpu())
    assert k().lookup_gradient(g, c.int(), n, out=got, accumulate=True) is got
    assert_close(got, 2 * want.cpu(), (2 * ((most + 2) * wide_half_step(t) * size + rounding(t, want)) + 2 * wide_half_step(t) * size + rounding(t, 2 * want)).cpu())


@gpu
@pytest.mark.parametrize("n", [262143, 262144, 300007, 150000001])
@pytest.mark.parametrize("rows", [3000, 6000, 140001])
def test_lookup_gradient_of_large_tables(rows, n):
    """Sorts of two, three and four digits, by comparison, by a cluster and by launches; what no code names is zero."""
    m = 4 if n < 1000000 else 1
    g = values((rows, m), F32, 75).cuda()
    c = torch.from_numpy(np.random.default_rng(76).integers(-5, n + 5, (rows, 1))).cuda()
    c[:: 7] = n - 1
    c[3:: 7] = 0
    got = k().lookup_gradient(g, c, n)
    named, place = torch.unique(c.flatten(), return_inverse=True)
    inside = (named >= 0) & (named < n)
    want, size, most = gradient_by_torch(g, place[:, None], len(named))
    assert_close(got[named[inside]], want[inside].cpu(), ((most + 2) * 2.0 ** -24 * size + rounding(F32, want))[inside].cpu())
    got[named[inside]] = 0
    assert not got.any()


@gpu
def test_lookup_gradient_against_differences():
    """The derivative of a weighted sum of lookups, by central differences in float64: the operator is linear, so they are
    off by rounding alone (a dozen terms, steps of one)."""
    rows, length, n, m = 6, 4, 9, 5
    w, c = values((n, m), F64, 1).cuda(), codes_of("absent", rows, length, n, 2, torch.int64).cuda()
    v = values((rows, m), F64, 3).cuda()
    g = k().lookup_gradient(v, c, n, 1.5)
    for i in range(n):
        for j in range(m):
            e = torch.zeros_like(w)
            e[i, j] = 1
            d = ((k().lookup(w + e, c, 1.5) - k().lookup(w - e, c, 1.5)) * v).sum() / 2
            assert abs(float(d - g[i, j])) <= 1e-12


@gpu
def test_lookup_of_nothing():
    w = values((5, 6), F32, 1).cuda()
    assert k().lookup(w, torch.empty((0, 3), dtype=torch.int64, device="cuda")).shape == (0, 6)
    assert not k().lookup(w, torch.empty((4, 0), dtype=torch.int32, device="cuda")).any()
    g = torch.ones((4, 6), device="cuda")
    assert not k().lookup_gradient(g, torch.empty((4, 0), dtype=torch.int64, device="cuda"), 5).any()
    assert not k().lookup_gradient(g[:0], torch.empty((0, 3), dtype=torch.int64, device="cuda"), 5).any()
    out = torch.ones((5, 6), device="cuda")
    k().lookup_gradient(g, torch.full((4, 2), -1, device="cuda"), 5, out=out, accumulate=True)
    assert bool((out == 1).all())
    k().lookup_gradient(g, torch.full((4, 2), -1, device="cuda"), 5, out=out)
    assert not out.any()


@gpu
@pytest.mark.parametrize("t,m", [(F32, 8), (BF16, 16), (BF16, 6), (F64, 3)])
def test_lookup_leaves_what_lies_around_its_results(t, m):
    rows, n = 37, 23
    w, c = values((n, m), t, 1).cuda(), codes_of("any", rows, 3, n, 2, torch.int64).cuda()
    g = values((rows, m), t, 3).cuda()
    room = torch.full((rows + n + 4, m), 7.0, dtype=t, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    code = {F32: 0, F64: 1, F16: 2, BF16: 3}[t]
    assert lib.sbb_lookup(code, w.data_ptr(), c.data_ptr(), 8, rows, 3, n, m, 1.0, room[1].data_ptr(), stream) == 0
    size = lib.sbb_lookup_gradient_workspace(code, rows, 3, n, m)
    work = torch.full((size + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    assert lib.sbb_lookup_gradient(code, g.data_ptr(), c.data_ptr(), 8, rows, 3, n, m, 1.0, 0, room[rows + 2].data_ptr(),
                                   work.data_ptr(), size, stream) == 0
    assert bool((room[[0, rows + 1, rows + n + 2, rows + n + 3]] == 7).all())
    assert bool((work[size:] == 0xA5).all())
    assert torch.equal(room[1:rows + 1], k().lookup(w, c))
    assert torch.equal(room[rows + 2:rows + 2 + n], k().lookup_gradient(g, c, n))


# ---- sampling --------------------------------------------------------------

SAMPLES = [  # rows, hypercolumns, units, spread of the support
    (1, 1, 1, 1.0), (3, 2, 2, 1.0), (5, 3, 10, 3.0), (9, 4, 33, 2.0), (4, 30, 100, 3.0), (2, 3, 128, 0.0), (2, 3, 300, 1.0),
    (2, 1, 513, 2.0), (2, 2, 1025, 0.5), (2, 1, 5000, 3.0), (1, 1, 40001, 3.0), (2, 1, 20000, 0.0), (1, 1, 70000, 0.05),
    (80, 2, 611, 2.0), (170, 1, 2051, 0.1), (300, 1, 1024, 3.0),   # as many as SMs: a block each
    (150, 2, 513, 0.1), (3, 1, 1024, 0.0), (600, 1, 8001, 2.0), (300, 2, 5000, 0.0), (150, 1, 8001, 0.5),
]
SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.6), dict(min_p=0.1), dict(temperature=0.5, top_k=7, top_p=0.8, min_p=0.02),
            dict(temperature=2.0, top_p=0.97), dict(top_k=400, top_p=0.999), dict(top_p=0.0), dict(top_k=1), dict(min_p=1.0)]


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,h,mc,spread", SAMPLES)
def test_sample(rows, h, mc, spread, t):
    rng = np.random.default_rng(rows * 1000 + mc)
    x = values((rows, h * mc), t, 7, spread)
    for i, how in enumerate(SETTINGS if mc <= 5000 else SETTINGS[5:8]):
        how = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **how}
        u = torch.from_numpy(rng.random((rows, h)).astype(np.float32))
        want = plain_sample_fast(x, h, mc, u, **how)
        got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), **how)
        assert got.dtype == torch.int64
        assert torch.equal(got.cpu(), want), (how, i)


def plain_sample_fast(x, h, mc, random, temperature, top_k, top_p, min_p):
    """:func:`plain_sample` without its quadratic sums: running sums in 64 bits."""
    rows = x.shape[0]
    x = x.double().numpy().reshape(rows, h, mc)
    pick = lambda v, r: float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))   # (numbers are rounded to float32)
    out = np.full((rows, h), -1, dtype=np.int64)
    for r in range(rows):
        t, k_, p, low = pick(temperature, r), int(pick(top_k, r)), pick(top_p, r), min(pick(min_p, r), 1.0)
        for g in range(h):
            v = np.where(np.isnan(x[r, g]), -np.inf, x[r, g])
            best = v.max()
            if best == -np.inf:
                continue
            with np.errstate(over="ignore", invalid="ignore"):
                w = np.where(v == best, 1.0, np.exp((v - best) / (t if t > 0 else 1.0)))
            order = np.argsort(-v, kind="stable")
            k_here = 1 if not t > 0 else k_
            if k_here > 0:
                order = order[:k_here]
            c = np.cumsum(w[order])
            before = np.concatenate(([0.0], c[:-1]))
            keep = (before < p * c[-1]) | (p >= 1)
            keep[0] = True
            order = order[keep]
            order = np.sort(order[(w[order] >= low) | (v[order] == best)])
            c = np.cumsum(w[order])
            at = np.flatnonzero(c > float(random[r, g]) * c[-1])
            last = np.flatnonzero(w[order] > 0)[-1]
            out[r, g] = g * mc + order[at[0] if len(at) else last]
    return torch.from_numpy(out)


def test_plain_sampling_two_ways():
    rng = np.random.default_rng(0)
    for mc, spread in ((1, 1.0), (9, 2.0), (40, 0.0)):
        x = values((3, 2 * mc), F32, 1, spread)
        for how in SETTINGS:
            how = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **how}
            u = torch.from_numpy(rng.random((3, 2)).astype(np.float32))
            assert torch.equal(plain_sample(x, 2, mc, u, **how), plain_sample_fast(x, 2, mc, u, **how))


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("mc", [5, 64, 200, 3001])
def test_sample_masks(mc, t):
    """-infinity, the type's lowest value, +infinity, NaN, all of a hypercolumn ruled out, equal values across the cut."""
    rows, h = 8, 2
    x = values((rows, h * mc), t, 11, 2.0)
    x[0] = -math.inf
    x[1, :mc] = -math.inf
    x[2, ::2] = -math.inf
    x[3, ::2] = torch.finfo(t).min
    x[4, 1::3] = math.nan
    x[5, 1::2] = math.inf
    x[6] = torch.round(x[6])
    x[7, mc:] = torch.finfo(t).min
    x[7, 0] = -0.0
    x[7, 1:mc] = 0.0
    rng = np.random.default_rng(mc)
    for how in SETTINGS:
        how = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **how}
        u = torch.from_numpy(rng.random((rows, h)).astype(np.float32))
        u[:, 0] = 0
        u[5, 1] = float(np.nextafter(np.float32(1), np.float32(0)))
        got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), **how).cpu()
        assert torch.equal(got, plain_sample_fast(x, h, mc, u, **how)), how
        assert bool((got[0] == -1).all()) and got[1, 0] == -1


@gpu
@pytest.mark.parametrize("rows,mc", [(16, 50), (16, 700), (16, 9000), (100, 1500)])
def test_sample_with_settings_of_each_row(rows, mc):
    h = 2
    x = values((rows, h * mc), BF16, 3, 3.0)
    rng = np.random.default_rng(5)
    u = torch.from_numpy(rng.random((rows, h)).astype(np.float32))
    temperature = torch.from_numpy(rng.uniform(0.2, 2, rows).astype(np.float32))
    temperature[::5] = 0
    top_k = torch.from_numpy(rng.integers(-1, 60, rows).astype(np.int32))
    top_p = torch.from_numpy(rng.uniform(0, 1.2, rows).astype(np.float32))
    min_p = torch.from_numpy(rng.uniform(0, 0.1, rows).astype(np.float32))
    got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), temperature.cuda(), top_k.cuda(), top_p.cuda(), min_p.cuda())
    assert torch.equal(got.cpu(), plain_sample_fast(x, h, mc, u, temperature, top_k, top_p, min_p))
    got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), 0.9, top_k.cuda(), 0.9, min_p.cuda())
    assert torch.equal(got.cpu(), plain_sample_fast(x, h, mc, u, 0.9, top_k, 0.9, min_p))
    every = lambda v: torch.full((rows,), v, device="cuda")   # a number and the same for every row
    assert torch.equal(k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), 0.7, 9, 0.95, 0.01),
                       k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), every(0.7), every(9).int(), every(0.95), every(0.01)))


def own_settings(rows, rng):
    """Settings of every row: temperatures, some of them 0, top-k, some of them none, top-p, min-p."""
    temperature = torch.from_numpy(rng.uniform(0.2, 2, rows).astype(np.float32))
    temperature[::5] = 0
    top_k = torch.from_numpy(rng.integers(-1, 60, rows).astype(np.int32))
    top_k[1::3] = 0
    return temperature, top_k, torch.from_numpy(rng.uniform(0.5, 1.1, rows).astype(np.float32)), torch.from_numpy(rng.uniform(0, 0.1, rows).astype(np.float32))


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,h,mc", [(700, 30, 10), (400, 30, 50), (700, 30, 100), (509, 31, 200), (400, 30, 401), (200, 30, 900)])
def test_sample_of_more_groups_than_warps(rows, h, mc, t):
    """A warp takes one hypercolumn after another, and each the settings of its own row."""
    x = values((rows, h * mc), t, 66, 2.0)
    rng = np.random.default_rng(67)
    u = torch.from_numpy(rng.random((rows, h)).astype(np.float32))
    u[::9] = small_numbers((len(u[::9]), h), 68)
    how = own_settings(rows, rng)
    got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), *[a.cuda() for a in how])
    assert torch.equal(got.cpu(), plain_sample_fast(x, h, mc, u, *how))
    assert torch.equal(k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), top_p=0.9).cpu(), plain_sample_fast(x, h, mc, u, 1.0, 0, 0.9, 0.0))


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,mc", [(148, 8193), (295, 9001), (160, 20000), (150, 50001), (296, 9001)])
def test_sample_wide_batches_with_settings_of_each_row(rows, mc, t):
    """Two blocks to a row, which read their parts from memory (from 296 rows on, one)."""
    x = values((rows, mc), t, 69, 2.0)
    x[2::4, ::3] = -math.inf
    x[3] = -math.inf
    rng = np.random.default_rng(70)
    u = torch.from_numpy(rng.random((rows, 1)).astype(np.float32))
    u[::9] = small_numbers((len(u[::9]), 1), 71)
    how = own_settings(rows, rng)
    assert torch.equal(k().sample_minicolumns(x.cuda(), 1, mc, u.cuda(), *[a.cuda() for a in how]).cpu(), plain_sample_fast(x, 1, mc, u, *how))
    assert torch.equal(k().sample_minicolumns(offset(x), 1, mc, u.cuda(), 1.0, how[1].cuda(), 0.95).cpu(), plain_sample_fast(x, 1, mc, u, 1.0, how[1], 0.95, 0.0))


@gpu
@pytest.mark.parametrize("rows,mc", [(8, 60), (8, 2000), (160, 2000)])
def test_sample_settings_of_a_row_out_of_range(rows, mc):
    """They act as the nearest in range: a temperature below 0 as 0, an infinite one as the limit (all that may be drawn is equally
    likely), a top-p below 0 as 0 and above 1 as 1, a min-p below 0 as 0 and above 1 as 1."""
    x = values((rows, mc), F32, 13, 2.0)
    x[:, 3::4] = -math.inf
    u = torch.from_numpy(np.random.default_rng(6).random((rows, 1)).astype(np.float32))
    column = lambda *v: torch.tensor(v, dtype=F32).repeat(rows // len(v))
    draw = lambda t, p, low, kk=0: k().sample_minicolumns(x.cuda(), 1, mc, u.cuda(), column(*t).cuda(), kk, column(*p).cuda(), column(*low).cuda()).cpu()
    for kk in (0, 9):
        got = draw((-1.0, 1.0, 1.0, 1.0), (1.0, -0.5, 1.0, 7.0), (0.0, 0.0, -3.0, 5.0), kk)
        want = draw((0.0, 1.0, 1.0, 1.0), (1.0, 0.0, 1.0, 1.0), (0.0, 0.0, 0.0, 1.0), kk)
        assert torch.equal(got, want)
        assert torch.equal(want, plain_sample_fast(x, 1, mc, u, column(0.0, 1.0, 1.0, 1.0), kk, column(1.0, 0.0, 1.0, 1.0), column(0.0, 0.0, 0.0, 1.0)))
    got = draw((math.inf, math.inf), (1.0, 0.5), (0.0, 0.0))
    drawn = x.gather(1, got)
    assert bool((drawn > -math.inf).all())
    flat = torch.where(x > -math.inf, 0.0, x.double()).to(F32)
    for r in range(0, rows, 2):
        assert torch.equal(got[r], plain_sample_fast(flat[r:r + 1], 1, mc, u[r:r + 1], 1.0, 0, 1.0, 0.0)[0])


@gpu
@pytest.mark.parametrize("mc", [37, 2500])
def test_sample_random_numbers_out_of_range(mc):
    x = values((1, mc), F32, 3).cuda()
    last = mc - 1
    for u, want in ((1.0, last), (5.0, last), (-3.0, 0), (math.nan, 0)):
        assert int(k().sample_minicolumns(x, 1, mc, torch.tensor([[u]], device="cuda"))) == want


def small_numbers(shape, seed):
    """Random numbers spread over the logarithm of what float32 holds above 0, and zeros."""
    rng = np.random.default_rng(seed)
    u = np.float32(2.0) ** rng.uniform(-149, 0, shape).astype(np.float32)
    u[rng.random(shape) < 0.25] = 0
    return torch.from_numpy(u.astype(np.float32).clip(0, np.nextafter(np.float32(1), np.float32(0))))


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,h,mc", [(40, 3, 2), (40, 3, 40), (40, 2, 300), (30, 1, 700), (30, 1, 3001), (20, 1, 20011), (160, 1, 2049), (600, 1, 1500)])
def test_sample_small_random_numbers(rows, h, mc, t):
    """A small random number falls to the units in front, however little they weigh: weights down to e^-700 of the largest, and some
    that are 0 in 64 bits.  (The plain form's running sums from the front are exact to n 2^-53 of themselves.)"""
    x = values((rows, h, mc), t, 61, 2.0)
    rng = np.random.default_rng(62)
    below = torch.from_numpy(rng.choice([0.0, 15, 30, 60, 100, 250, 700, 1500], (rows, h, 1)))
    first = torch.from_numpy(rng.integers(1, mc, (rows, h, 1)))
    x = torch.where(torch.arange(mc) < first, (x.double() - below).to(t), x).reshape(rows, h * mc)
    u = small_numbers((rows, h), 63)
    for how in (dict(), dict(top_k=mc // 2 + 1), dict(top_k=mc), dict(min_p=1e-20), dict(temperature=0.5, min_p=1e-12), dict(top_k=3, top_p=0.9),
                dict(top_p=0.99), dict(temperature=7.0, top_k=300)):
        how = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **how}
        got = k().sample_minicolumns(x.cuda(), h, mc, u.cuda(), **how).cpu()
        assert torch.equal(got, plain_sample_fast(x, h, mc, u, **how)), how
    assert int(k().sample_minicolumns(torch.tensor([[-60.0, 0.0]], dtype=t).cuda(), 1, 2, torch.zeros((1, 1)).cuda())) == 0


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,mc", [(2, 200001), (150, 20001), (9, 700)])
def test_sample_small_random_numbers_behind_a_mask(rows, mc, t):
    """The first unit that may be drawn stands far behind: those in front are masked, or too light for 64 bits."""
    x = values((rows, mc), t, 64, 2.0)
    x[:, :mc // 3] = -math.inf
    x[:, mc // 3:mc // 2] -= 2000
    x[0, :mc - 1] = -math.inf
    u = torch.zeros((rows, 1))
    u[1::2] = 1e-30
    for how in (dict(), dict(top_k=mc - 5), dict(min_p=1e-3)):
        how = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **how}
        got = k().sample_minicolumns(x.cuda(), 1, mc, u.cuda(), **how).cpu()
        assert torch.equal(got, plain_sample_fast(x, 1, mc, u, **how)), how
        assert int(got[0]) == mc - 1


@gpu
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("mc", [32, 61, 127, 256, 512, 1000, 1024])
def test_sample_random_numbers_at_the_borders(mc, t):
    """The floats around every border of two units (which sums in 32 bits do not tell apart), of nearly equal weights, so that
    roundings add up, and of spread ones."""
    for spread, top_p in ((0.0, 1.0), (1e-3, 1.0), (1.0, 1.0), (0.01, 0.7)):
        x = values((1, mc), t, 65, spread)
        w = torch.exp(x.double() - x.double().max())[0]
        if top_p < 1:
            order = torch.sort(w, descending=True, stable=True).indices
            c = w[order].cumsum(0)
            out = order[(c - w[order]) >= float(np.float32(top_p)) * c[-1]]
            w[out] = 0
        border = (w.cumsum(0) / w.sum()).numpy().astype(np.float32)
        u = np.concatenate([border, np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(1))]).clip(0, np.nextafter(np.float32(1), np.float32(0)))
        u = torch.from_numpy(u)[:, None]
        rows = x.expand(u.shape[0], mc)
        got = k().sample_minicolumns(rows.cuda(), 1, mc, u.cuda(), top_p=top_p).cpu()
        assert torch.equal(got, plain_sample_fast(rows, 1, mc, u, 1.0, 0, top_p, 0.0)), spread


def offset(a):
    """The same values one element behind a boundary of 16 bytes and more."""
    b = torch.empty(a.numel() + 1, dtype=a.dtype, device="cuda")[1:].view(a.shape)
    b.copy_(a)
    assert b.is_contiguous() and b.data_ptr() % 16 == a.element_size() % 16
    return b


@gpu
@pytest.mark.parametrize("t", ALL)
def test_operators_on_tensors_that_begin_anywhere(t):
    for rows, mc in ((3, 40), (2, 200), (3, 4096), (160, 1033)):
        x = values((rows, mc), t, 51, 2.0)
        u = torch.from_numpy(np.random.default_rng(52).random((rows, 1)).astype(np.float32))
        for how in (dict(temperature=1.0, top_k=20, top_p=0.9, min_p=0.0), dict(temperature=1.0, top_k=0, top_p=0.9, min_p=0.01),
                    dict(temperature=0.0, top_k=0, top_p=1.0, min_p=0.0)):
            assert torch.equal(k().sample_minicolumns(offset(x), 1, mc, offset(u), **how).cpu(), plain_sample_fast(x, 1, mc, u, **how))
        units, teacher = teacher_of(x, 1, mc, 7, 53)
        want = k().distill_gradient(x.cuda(), 1, mc, units.cuda(), teacher.cuda(), 2.0)
        _, grad, loss_off, grad_off = plain_distill(x, 1, mc, units, teacher, 2.0, None)
        got = k().distill_gradient(offset(x), 1, mc, offset(units), offset(teacher), 2.0)
        assert_close(got[0], want[0].double().cpu(), 2 * loss_off)
        assert_close(got[1], grad, grad_off + rounding(t, grad))
    w, c = values((31, 48), t, 54), codes_of("absent", 20, 5, 31, 55, torch.int64)
    assert torch.equal(k().lookup(offset(w), offset(c)), k().lookup(w.cuda(), c.cuda()))
    g = values((20, 48), t, 56)
    want, size, most = plain_gradient(g, c, 31, 1.0)
    assert_close(k().lookup_gradient(offset(g), offset(c), 31), want, (most + 2) * wide_half_step(t) * size + rounding(t, want))


@gpu
def test_sample_frequencies_are_the_softmax():
    """Equally spaced random numbers: every unit is drawn as often as its part of the interval says, to one draw at either end."""
    mc, draws = 23, 4096
    x = values((1, mc), F32, 9, 1.5)
    u = ((torch.arange(draws) + 0.5) / draws)[:, None]
    got = k().sample_minicolumns(x.expand(draws, mc).cuda(), 1, mc, u.cuda()).cpu().flatten()
    part = torch.softmax(x.double()[0], 0) * draws
    assert bool(((torch.bincount(got, minlength=mc) - part).abs() <= 1).all())


@gpu
def test_sample_of_nothing():
    assert k().sample_minicolumns(torch.empty((0, 12), device="cuda"), 3, 4, torch.empty((0, 3), device="cuda")).shape == (0, 3)


# ---- distillation ----------------------------------------------------------

DISTILLS = [  # rows, hypercolumns, units, kept, temperature
    (1, 1, 1, 1, 1.0), (3, 2, 2, 1, 2.0), (4, 1, 10, 3, 2.0), (3, 30, 100, 5, 1.0), (2, 3, 129, 8, 0.5), (2, 2, 300, 300, 4.0),
    (3, 1, 1025, 64, 1.0), (2, 1, 5003, 32, 3.0), (1, 2, 20000, 70, 1.0), (1, 1, 60000, 16, 1.0), (5, 7, 31, 40, 1.0),
    (1, 1, 600, 700, 2.0), (1, 1, 3001, 1500, 1.0),   # more kept units than a block has threads
    (400, 1, 5003, 200, 1.0), (150, 1, 8192, 5, 2.0), (150, 1, 8193, 5, 2.0),
    (37, 5, 8, 3, 1.0), (11, 3, 9, 20, 2.0), (50, 3, 16, 16, 1.0), (7, 3, 33, 9, 1.0), (301, 7, 47, 10, 2.0), (5, 5, 64, 64, 1.0), (5, 5, 65, 40, 1.0),
]


def teacher_of(x, h, mc, kept, seed):
    t = x.double().reshape(x.shape[0], h, mc) + torch.from_numpy(np.random.default_rng(seed).standard_normal((x.shape[0], h, mc)))
    if kept > mc:   # more entries than units: some named twice, some absent
        units = torch.from_numpy(np.random.default_rng(seed).integers(-2, mc + 2, (x.shape[0], h, kept)))
        return units, t.gather(2, units.clamp(0, mc - 1)).to(x.dtype)
    v, units = t.topk(kept, dim=2)
    return units, v.to(x.dtype)


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,h,mc,kept,temperature", DISTILLS)
def test_distill(rows, h, mc, kept, temperature, t):
    x = values((rows, h * mc), t, 21, 3.0)
    units, teacher = teacher_of(x, h, mc, kept, 22)
    weight = torch.from_numpy(np.random.default_rng(1).uniform(0.5, 2, rows)).to(F64 if t == F64 else F32)
    if rows > 2:
        weight[1] = 0
    for w, index in ((None, torch.int64), (weight, torch.int32)):
        want, grad, loss_off, grad_off = plain_distill(x, h, mc, units, teacher, temperature, w)
        args = (x.cuda(), h, mc, units.to(index).cuda(), teacher.cuda(), temperature, None if w is None else w.cuda())
        loss, gradient = k().distill_gradient(*args)
        assert loss.dtype == weight.dtype and gradient.dtype == t
        assert_close(loss, want, loss_off)
        assert_close(gradient, grad, grad_off + rounding(t, grad))
        assert_close(k().distill_loss(*args), want, loss_off)


def distill_by_torch(x, units, teacher, temperature):
    """(loss, gradient, bound of the loss, bound of the gradient) of whole rows in 64 bits, as in :func:`plain_distill`; on the tensors' device.
    Entries out of range are absent; no row is without one."""
    u = wide_half_step(x.dtype)
    mc, kept = x.shape[1], units.shape[1]
    there = (units >= 0) & (units < mc)
    named = torch.where(there, units, 0)
    v, tv = x.double() / temperature, torch.where(there, teacher.double(), -math.inf) / temperature
    log_q, log_p = torch.log_softmax(v, 1), torch.log_softmax(tv, 1)
    p, of = log_p.exp(), log_q.gather(1, named)
    pp = torch.zeros_like(v).scatter_add_(1, named, p)
    span = max(float(v.max() - v.min()), float(tv[there].max() - tv[there].min()))
    c = (6 * span + mc + kept + 40) * u
    zero = torch.zeros_like(p)
    loss = temperature ** 2 * torch.where(p > 0, p * (log_p - of), zero).sum(1)
    loss_off = temperature ** 2 * torch.where(p > 0, p * (log_p.abs() + of.abs() + 1), zero).sum(1) * c
    q = log_q.exp()
    return loss, temperature * (q - pp), loss_off, temperature * (q + pp) * c + (1e-37 if x.dtype != F64 else 1e-300)


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,mc,kept,among", [(3, 600, 300000, 600), (2, 9001, 300000, 9001), (1, 60001, 300000, 60001), (2, 700, 300000, 3), (1, 700001, 5000, 700001),
                                                 (2, 8192, 129, 8192), (2, 8193, 513, 100), (3, 513, 128, 513)])
def test_distill_with_long_lists(rows, mc, kept, among, t):
    """Lists of more entries than a block has threads, most units named many times, some entries absent; within a time that their square
    would exceed by far (300000 entries in pieces of 128: 2344 x 300000 steps a thread)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(kept + mc)
    x = (torch.randn((rows, mc), generator=gen, device="cuda") * 2).to(t)
    units = torch.randint(-among // 8 - 1, among + among // 8 + 1, (rows, kept), generator=gen, device="cuda")
    units = torch.where(units < among, units, mc + units)   # (no unit from among on)
    teacher = (torch.randn((rows, kept), generator=gen, device="cuda") * 2).to(t)
    call = lambda: k().distill_gradient(x, 1, mc, units[:, None], teacher[:, None], 2.0)
    call()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    loss, gradient = call()
    end.record()
    end.synchronize()
    assert start.elapsed_time(end) < 300
    want, grad, loss_off, grad_off = distill_by_torch(x, units, teacher, 2.0)
    assert_close(loss[:, 0], want.cpu(), loss_off.cpu())
    assert_close(gradient, grad.cpu(), (grad_off + rounding(t, grad)).cpu())
    again, same = call()
    assert torch.equal(loss, again) and torch.equal(gradient, same)


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("rows,h,mc,kept", [(1009, 80, 10, 3), (1001, 80, 7, 9), (1000, 80, 100, 5), (503, 80, 200, 8), (500, 80, 300, 8), (251, 80, 400, 8), (250, 80, 511, 40)])
def test_distill_of_more_groups_than_lanes(rows, h, mc, kept, t):
    """Lanes take one hypercolumn after another, and each the weight of its own row."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(mc)
    x = (torch.randn((rows, h * mc), generator=gen, device="cuda") * 2).to(t)
    units = torch.randint(0, mc, (rows, h, kept), generator=gen, device="cuda")
    units[..., 1:][torch.rand(units[..., 1:].shape, generator=gen, device="cuda") < 0.2] = -1
    teacher = (torch.randn((rows, h, kept), generator=gen, device="cuda") * 2).to(t)
    weight = torch.rand(rows, generator=gen, device="cuda", dtype=F64).to(F64 if t == F64 else F32) + 0.5
    weight[::10] = 0
    loss, gradient = k().distill_gradient(x, h, mc, units, teacher, 2.0, weight)
    want, grad, loss_off, grad_off = distill_by_torch(x.view(-1, mc), units.view(-1, kept), teacher.view(-1, kept), 2.0)
    w = weight.double().repeat_interleave(h)
    assert_close(loss.flatten(), (want * w).cpu(), (loss_off * w).cpu())
    grad = grad * w[:, None]
    assert_close(gradient.view(-1, mc), grad.cpu(), (grad_off * w[:, None] + rounding(t, grad)).cpu())


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("mc", [6, 100, 700, 9000])
def test_distill_masks(mc, t):
    rows, h, kept = 10, 2, 4
    x = values((rows, h * mc), t, 31, 2.0)
    units, teacher = teacher_of(x, h, mc, kept, 32)
    x[0, :mc] = -math.inf                                # nothing in the student
    units[1, 1] = -1                                     # nothing kept
    units[2, :, 1:] = mc                                 # one kept
    teacher[3, 0] = -math.inf                            # a teacher that rules all out
    teacher[4, :, 0] = -math.inf                         # ... or one
    x[5].view(h, mc).scatter_(1, units[5, :, 3:], -math.inf)   # a kept unit that the student rules out: an infinite loss
    units[6, 0] = units[6, 0, :1].clone()                # the same unit four times
    x[7, ::2] = torch.finfo(t).min                       # the lowest value
    teacher[7, 1, 0] = torch.finfo(t).min
    x[8], teacher[8] = math.nan, math.nan                # behind a weight of zero
    units[9, 0, 2:] = units[9, 0, :2].clone()            # two units twice each
    weight = torch.ones(rows, dtype=F64 if t == F64 else F32)
    weight[8] = 0
    want, grad, loss_off, grad_off = plain_distill(x, h, mc, units, teacher, 1.5, weight)
    loss, gradient = k().distill_gradient(x.cuda(), h, mc, units.cuda(), teacher.cuda(), 1.5, weight.cuda())
    # row 7: p times the lowest value may lie beyond the largest float32 (6 units, float32: 3.4557e38 > 3.4028e38), which is an
    # infinite loss in float32
    want = want.to(loss.dtype).double()
    assert_close(loss, want, loss_off)
    assert_close(gradient, grad, grad_off + rounding(t, grad))
    assert torch.equal(loss, k().distill_loss(x.cuda(), h, mc, units.cuda(), teacher.cuda(), 1.5, weight.cuda()))
    assert bool(torch.isinf(loss[5]).all()) and float(loss[0, 0]) == 0 and not gradient[8].any() and not gradient[0, :mc].any()
    # a NaN of the student stays in its hypercolumn
    x[9, mc + 1] = math.nan
    loss, gradient = k().distill_gradient(x.cuda(), h, mc, units.cuda(), teacher.cuda(), 1.5, weight.cuda())
    assert bool(torch.isnan(loss[9, 1])) and bool(torch.isnan(gradient[9, mc:]).all())
    assert_close(loss[9, :1], want[9, :1], loss_off[9, :1])
    assert_close(gradient[9, :mc], grad[9, :mc], grad_off[9, :mc] + rounding(t, grad[9, :mc]))
    # ... also where there is nothing else, and one of the teacher's does too
    x[0, :mc] = math.nan
    teacher[3, 0, :] = math.nan
    loss, gradient = k().distill_gradient(x.cuda(), h, mc, units.cuda(), teacher.cuda(), 1.5, weight.cuda())
    assert bool(torch.isnan(loss[0, 0])) and bool(torch.isnan(gradient[0, :mc]).all())
    assert bool(torch.isnan(loss[3, 0])) and bool(torch.isnan(gradient[3, :mc]).any())


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("mc,kept", [(6, 2), (100, 3), (333, 40), (700, 4), (1025, 4), (9001, 600), (30001, 4)])
def test_distill_with_infinity(mc, kept, t):
    """exp(infinity - infinity) is not a number, and so is what is divided by it, wherever in the hypercolumn the infinity stands and
    wherever the tensor begins.  A teacher's reaches the loss and the units that it keeps."""
    x = values((5, mc), t, 81, 2.0)
    units, teacher = teacher_of(x, 1, mc, kept, 82)
    for j, at in enumerate((0, mc // 2, mc - 1)):
        x[j, at] = math.inf
    teacher[3, 0, kept // 2] = math.inf
    for place in (lambda a: a.cuda(), offset):
        loss, gradient = k().distill_gradient(place(x), 1, mc, units.cuda(), teacher.cuda(), 2.0)
        assert torch.equal(torch.isnan(loss.cpu()[:, 0]), torch.tensor([True, True, True, True, False]))
        named = torch.zeros(mc, dtype=torch.bool)
        named[units[3, 0]] = True
        gradient = gradient.cpu()
        assert bool(torch.isnan(gradient[:3]).all()) and torch.equal(torch.isnan(gradient[3]), named) and not torch.isnan(gradient[4]).any()
        again = k().distill_loss(place(x), 1, mc, units.cuda(), teacher.cuda(), 2.0)
        assert torch.equal(torch.isnan(again), torch.isnan(loss))


@gpu
@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("mc", [6, 100, 512, 700, 9000])
def test_distill_where_nothing_is_kept_beside_a_nan(mc, t):
    """Exactly 0 where the teacher keeps nothing or the student rules all out, whatever the other holds."""
    x = values((5, mc), t, 91, 2.0)
    units, teacher = teacher_of(x, 1, mc, 3, 92)
    x[0, mc // 2] = math.nan
    units[0] = -1
    x[1, 0] = math.nan
    teacher[1] = -math.inf
    x[2] = -math.inf
    teacher[2, 0, 1] = math.nan
    x[3, mc - 1] = math.inf
    teacher[3] = -math.inf
    loss, gradient = k().distill_gradient(x.cuda(), 1, mc, units.cuda(), teacher.cuda(), 2.0)
    assert bool((loss[:4] == 0).all()) and bool((gradient[:4] == 0).all()) and float(loss[4]) > 0
    assert torch.equal(loss, k().distill_loss(x.cuda(), 1, mc, units.cuda(), teacher.cuda(), 2.0))


@gpu
def test_distill_gradient_against_differences():
    """Central differences in float64 with steps of 1e-4: the loss's third derivative is below its temperature-scaled size of
    one, so they are off by at most 1e-8 and by 1e-16 / 1e-4 for the roundings."""
    rows, h, mc, kept = 2, 2, 7, 3
    x = values((rows, h * mc), F64, 41, 1.5)
    units, teacher = teacher_of(x, h, mc, kept, 42)
    weight = torch.tensor([0.75, 2.0], dtype=F64)
    rest = (h, mc, units.cuda(), teacher.cuda(), 2.0, weight.cuda())
    gradient = k().distill_gradient(x.cuda(), *rest)[1].cpu()
    for r in range(rows):
        for i in range(h * mc):
            e = torch.zeros_like(x)
            e[r, i] = 1e-4
            d = (k().distill_loss((x + e).cuda(), *rest) - k().distill_loss((x - e).cuda(), *rest)).sum() / 2e-4
            assert abs(float(d) - float(gradient[r, i])) <= 1e-7


@gpu
def test_distill_of_nothing():
    x = values((3, 8), F32, 1).cuda()
    none = torch.empty((3, 2, 0), dtype=torch.int64, device="cuda")
    loss, gradient = k().distill_gradient(x, 2, 4, none, none.float())
    assert loss.shape == (3, 2) and not loss.any() and not gradient.any()
    loss, gradient = k().distill_gradient(x[:0], 2, 4, none[:0], none[:0].float())
    assert loss.shape == (0, 2) and gradient.shape == (0, 8)


# ---- together, and how calls are made --------------------------------------

def chain(x, w, u, teacher_units, teacher, h, mc, n):
    """Codes drawn from a hidden layer, the support they give in the next one, its distance from a teacher, and the gradient
    of that with respect to the weights."""
    codes = k().sample_minicolumns(x, h, mc, u, temperature=0.9, top_k=20, top_p=0.95)
    support = k().lookup(w, codes, 0.5)
    loss, gradient = k().distill_gradient(support, 1, w.shape[1], teacher_units, teacher, 2.0)
    return codes, support, loss, k().lookup_gradient(gradient, codes, n, 0.5), k().sample_minicolumns(support, 1, w.shape[1], u[:, :1].contiguous())


def chain_inputs(t, rows=24, h=5, mc=40, m=33, kept=4, seed=0):
    n = h * mc
    x, w = values((rows, n), t, seed + 1, 3.0), values((n, m), t, seed + 2)
    u = torch.from_numpy(np.random.default_rng(seed + 3).random((rows, h)).astype(np.float32))
    units, teacher = teacher_of(values((rows, m), t, seed + 4, 2.0), 1, m, kept, seed + 5)
    return [a.cuda() for a in (x, w, u, units, teacher)] + [h, mc, n]


@gpu
@pytest.mark.parametrize("t", ALL)
def test_operators_together(t):
    x, w, u, units, teacher, h, mc, n = args = chain_inputs(t)
    codes, support, loss, grad, answer = chain(*args)
    cpu = [a.cpu() for a in (x, w, u, units, teacher, codes, support, grad)]
    assert torch.equal(cpu[5], plain_sample_fast(cpu[0], h, mc, cpu[2], 0.9, 20, 0.95, 0.0))
    want, size = plain_lookup(cpu[1], cpu[5], 0.5)
    assert_close(support, want, (h + 2) * wide_half_step(t) * size + rounding(t, want))
    _, g, _, g_off = plain_distill(cpu[6], 1, w.shape[1], cpu[3], cpu[4], 2.0, None)
    back, back_size, most = plain_gradient(g, cpu[5], n, 0.5)
    slack, _, _ = plain_gradient(g_off + rounding(t, g), cpu[5], n, 0.5)
    assert_close(grad, back, slack + (most + 2) * wide_half_step(t) * (back_size + slack) + rounding(t, back.abs() + slack))
    assert torch.equal(answer.cpu(), plain_sample_fast(cpu[6], 1, w.shape[1], cpu[2][:, :1], 1.0, 0, 1.0, 0.0))


@gpu
def test_operators_captured_into_a_graph():
    args, other = chain_inputs(F32), chain_inputs(F32, seed=100)
    want = chain(*other)
    tensors = args[:5]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(*args)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(*args)
    with torch.cuda.graph(second):
        got2 = chain(*args)
    for a, b in zip(tensors, other[:5]):
        a.copy_(b)
    graph.replay()
    second.replay()
    graph.replay()
    for a, b, c in zip(got, got2, want):
        assert torch.equal(a, c) and torch.equal(b, c)
    # ... and the ways that large calls take
    rows, n, m = 6000, 300, 24
    g, c, x = values((rows, m), F32, 1).cuda(), codes_of("few", rows, 1, n, 2, torch.int64).cuda(), values((200, 3000), BF16, 3, 3.0).cuda()
    u = torch.rand((200, 1), device="cuda")
    large = lambda: (k().lookup_gradient(g, c, n), k().lookup_gradient(g.repeat(30, 1)[:140000], c.repeat(30, 1)[:140000], n),
                     k().sample_minicolumns(x, 1, 3000, u, top_p=0.9), k().sample_minicolumns(x[:2], 1, 3000, u[:2], top_k=40),
                     *k().distill_gradient(x, 1, 3000, c[:200, None, :1], x[:, None, :1].contiguous(), 1.0))
    want = large()
    third = torch.cuda.CUDAGraph()
    with torch.cuda.graph(third):
        got = large()
    third.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_operators_on_several_streams_at_once():
    sets = [chain_inputs(t, rows=200, seed=10 * i) for i, t in enumerate((F32, BF16, F64, F16))]
    want = [chain(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(5):
        for i, (s, a) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(chain(*a))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for one in g:
            assert all(torch.equal(a, b) for a, b in zip(one, w))


@gpu
def test_operators_copy_what_is_not_contiguous():
    x, w, u, units, teacher, h, mc, n = args = chain_inputs(F32)
    want = chain(*args)
    wide = lambda a: torch.stack((a, a), dim=a.dim()).movedim(-1, 0)[1]
    strided = [wide(a) for a in args[:5]]
    assert not any(a.is_contiguous() for a in strided)
    assert all(torch.equal(a, b) for a, b in zip(chain(*strided, h, mc, n), want))


@gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("n,h,mc", [(40, 5, 12), (300, 3, 100), (64, 1, 10)])
def test_layers_take_codes(n, h, mc, dtype):
    """A layer's activation from codes and from the dense row they stand for; the units drawn are the sampler's of its support,
    and feed the next layer.  Both sum n products: 2 (n + 8) roundings of the magnitudes they add, through a softmax, whose
    derivative is at most a half, and whose own roundings are a dozen."""
    from streambrain_b200.backend.b200_backend import DenseLayer, StructuralPlasticityLayer
    np.random.seed(1)
    hidden = StructuralPlasticityLayer(n, h, mc, 0.01, -100.0, 0.05, 0.02, 0.5, 16, (1, 1 / mc, 1 / mc), dtype=dtype)
    out = DenseLayer(h * mc, 1, 10, 0.01, (0.1, 0.1, 0.01), dtype=dtype)
    rng = np.random.default_rng(2)
    x = (rng.random((33, n)) < 0.3).astype(dtype)
    length = int(x.sum(1).max())
    codes = np.full((33, length), -1, dtype=np.int64)
    for r in range(33):
        codes[r, :int(x[r].sum())] = np.flatnonzero(x[r])
    t = F32 if dtype is np.float32 else F64
    u = half_step(t)
    c = torch.from_numpy(codes).cuda()
    want = hidden.compute_activation(torch.from_numpy(x).cuda())
    size = float((x @ np.abs(hidden.weights)).max()) + float(np.abs(hidden.bias).max())
    bound = (2 * (n + 8) * size + 24) * u
    for index in (torch.int64, torch.int32):
        got = hidden.compute_activation(c.to(index))
        assert got.dtype == t and float((got - want).abs().max()) <= bound
    random = torch.from_numpy(rng.random((33, h)).astype(np.float32)).cuda()
    units = hidden.sample_units(c, random, temperature=0.8, top_p=0.9)
    support = k().lookup(hidden.state_tensor("weights"), c) + hidden.state_tensor("bias")
    assert torch.equal(units, k().sample_minicolumns(support, h, mc, random, temperature=0.8, top_p=0.9))
    assert out.compute_activation(units).shape == (33, 10)
    with pytest.raises(TypeError):
        hidden.compute_activation(torch.from_numpy(codes))
    with pytest.raises(TypeError):
        hidden.compute_activation(c[0])


# ---- refusals (no device needed) -------------------------------------------

class _Codes:
    """What a layer asks of a tensor of codes on CUDA device ``device``, without the device."""
    is_cuda, dtype, shape = True, torch.int64, (2, 3)

    def __init__(self, device):
        self.device, self._number = torch.device("cpu"), device

    def dim(self):
        return 2

    def get_device(self):
        return self._number

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096

    def element_size(self):
        return 8


def test_layers_refuse_codes_of_another_device(monkeypatch):
    from types import SimpleNamespace

    from streambrain_b200.backend import b200_backend as b
    layer = b.DenseLayer.__new__(b.DenseLayer)
    layer.out_features, layer._tdtype, layer._handle, layer.hypercolumns, layer.minicolumns = 4, F32, None, 2, 2
    calls = []
    monkeypatch.setattr(b, "_current_device", lambda: 1)
    monkeypatch.setattr(b, "_stream_ptr", lambda: 0)
    monkeypatch.setattr(b, "lib", SimpleNamespace(sbb_layer_forward_codes=lambda *a: calls.append(a) or 0))
    for call in (lambda c: layer._forward_codes(c, 1), lambda c: layer.sample_units(c, None)):
        with pytest.raises(ValueError):
            call(_Codes(0))
    assert not calls
    assert layer._forward_codes(_Codes(1), 1).shape == (2, 4) and len(calls) == 1


def test_wrappers_refuse_host_tensors_and_wrong_types():
    pytest.importorskip("streambrain_b200.kernels_device")
    w, c = torch.zeros((4, 3)), torch.zeros((2, 1), dtype=torch.int64)
    for call in (lambda: k().lookup(w, c), lambda: k().lookup_gradient(w, c, 4), lambda: k().lookup(w.numpy(), c),
                 lambda: k().sample_minicolumns(w, 1, 3, w[:, :1]), lambda: k().distill_loss(w, 1, 3, c[..., None], w[..., None])):
        with pytest.raises(TypeError):
            call()


@gpu
def test_wrappers_refuse():
    f = lambda *shape, t=F32: torch.zeros(shape, dtype=t, device="cuda")
    i = lambda *shape: torch.zeros(shape, dtype=torch.int64, device="cuda")
    bad = [
        (TypeError, lambda: k().lookup(f(4, 3), f(2, 1))),
        (TypeError, lambda: k().lookup(i(4, 3), i(2, 1))),
        (TypeError, lambda: k().lookup(f(4, 3), torch.zeros((2, 1), dtype=torch.int64))),
        (ValueError, lambda: k().lookup(f(4, 3), i(2))),
        (ValueError, lambda: k().lookup(f(4), i(2, 1))),
        (_lib.SbbError, lambda: k().lookup(f(0, 3), i(2, 1))),
        (ValueError, lambda: k().lookup_gradient(f(3, 3), i(2, 1), 4)),
        (ValueError, lambda: k().lookup_gradient(f(2, 3), i(2, 1), 0)),
        (ValueError, lambda: k().lookup_gradient(f(2, 3), i(2, 1), 4, accumulate=True)),
        (ValueError, lambda: k().lookup_gradient(f(2, 3), i(2, 1), 4, out=f(5, 3))),
        (ValueError, lambda: k().lookup_gradient(f(2, 3), i(2, 1), 4, out=f(3, 4).t())),
        (TypeError, lambda: k().lookup_gradient(f(2, 3), i(2, 1), 4, out=f(4, 3, t=F64))),
        (ValueError, lambda: k().sample_minicolumns(f(2, 6), 2, 4, f(2, 2))),
        (ValueError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 1))),
        (TypeError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2, t=F64))),
        (TypeError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), top_k=f(2))),
        (ValueError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), top_p=f(3))),
        (_lib.SbbError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), temperature=-1.0)),
        (_lib.SbbError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), temperature=math.nan)),
        (_lib.SbbError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), min_p=1.5)),
        (_lib.SbbError, lambda: k().sample_minicolumns(f(2, 6), 2, 3, f(2, 2), top_p=-0.5)),
        (ValueError, lambda: k().distill_loss(f(2, 6), 2, 4, i(2, 2, 1), f(2, 2, 1))),
        (ValueError, lambda: k().distill_loss(f(2, 6), 2, 3, i(2, 2, 1), f(2, 2, 2))),
        (TypeError, lambda: k().distill_loss(f(2, 6), 2, 3, i(2, 2, 1), f(2, 2, 1, t=F16))),
        (TypeError, lambda: k().distill_loss(f(2, 6), 2, 3, i(2, 2, 1), f(2, 2, 1), weight=f(2, t=F64))),
        (ValueError, lambda: k().distill_loss(f(2, 6), 2, 3, i(2, 2, 1), f(2, 2, 1), weight=f(3))),
        (_lib.SbbError, lambda: k().distill_gradient(f(2, 6), 2, 3, i(2, 2, 1), f(2, 2, 1), temperature=0.0)),
    ]
    for j, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail("call %d went through" % j)


def test_layers_refuse_dense_rows_of_integers(monkeypatch):
    """An integer tensor of a dense row's shape is refused, as it was before layers took codes, unless it is said to hold codes."""
    from streambrain_b200.backend import b200_backend as b
    layer = b.DenseLayer.__new__(b.DenseLayer)
    layer.in_features, layer._handle, layer.dtype, layer._tdtype, calls = 6, None, np.float32, F32, []
    monkeypatch.setattr(layer, "_forward_codes", lambda c, softmax: calls.append(c.shape), raising=False)
    for t in (torch.int32, torch.int64):
        with pytest.raises(TypeError):
            layer.compute_activation(torch.zeros((2, 6), dtype=t))
    assert not calls
    layer.compute_activation(torch.zeros((2, 6), dtype=torch.int64), codes=True)
    layer.compute_activation(torch.zeros((2, 5), dtype=torch.int64))
    layer.compute_activation(torch.zeros((2, 5), dtype=torch.int32), codes=True)
    assert calls == [(2, 6), (2, 5), (2, 5)]
    for other in (torch.zeros((2, 6)), np.zeros((2, 6), dtype=np.int64)):
        with pytest.raises(TypeError):
            layer.compute_activation(other, codes=True)


def test_warp_collectives_stay_where_they_are():
    """An asm statement that is not volatile may be moved into a branch that not all lanes take; one that waits for all of them may not."""
    import pathlib
    import re
    sources = [f for f in (pathlib.Path(_lib.__file__).parent / "csrc").iterdir() if f.suffix in (".cu", ".cuh", ".h")]
    assert sources
    for f in sources:
        for m in re.finditer(r"\basm\s*(volatile)?\s*\(\s*\"([^\"]*)", f.read_text()):
            assert m.group(1) or not re.search(r"\b(redux|shfl|vote|match|bar|barrier|activemask)\.", m.group(2)), (f.name, m.group(2))


def test_entries_from_many_threads():
    """(Without rows nothing is launched.)"""
    from concurrent.futures import ThreadPoolExecutor
    at, how = ctypes.c_void_p(4096), _lib.Sampling(1.0, 1.0, 0.0, 0)
    want = 0 if lib.sbb_device_count() > 0 else _lib.ERR_NO_DEVICE

    def calls(_):
        return (lib.sbb_lookup(0, at, at, 8, 0, 1, 4, 3, 1.0, at, None), lib.sbb_sample_minicolumns(0, at, at, 0, 1, 3, ctypes.byref(how), at, None),
                lib.sbb_distill(0, at, at, 8, at, None, 0, 1, 3, 1, 1.0, at, at, None), lib.sbb_lookup(7, at, at, 8, 0, 1, 4, 3, 1.0, at, None))

    with ThreadPoolExecutor(16) as pool:
        assert set(pool.map(calls, range(400))) == {(want, want, want, _lib.ERR_INVALID)}


def test_entries_refuse_before_any_device_work():
    at, big = ctypes.c_void_p(4096), 1 << 40
    how = _lib.Sampling(1.0, 1.0, 0.0, 0)
    look = lambda **a: lib.sbb_lookup(*[{**dict(dtype=0, w=at, c=at, bytes=8, rows=2, l=1, n=4, m=3, scale=1.0, out=at, stream=None), **a}[x]
                                        for x in ("dtype", "w", "c", "bytes", "rows", "l", "n", "m", "scale", "out", "stream")])
    grad = lambda **a: lib.sbb_lookup_gradient(*[{**dict(dtype=0, g=at, c=at, bytes=8, rows=2, l=1, n=4, m=3, scale=1.0, add=0, out=at, work=at,
                                                            size=1 << 30, stream=None), **a}[x] for x in (
        "dtype", "g", "c", "bytes", "rows", "l", "n", "m", "scale", "add", "out", "work", "size", "stream")])
    draw = lambda **a: lib.sbb_sample_minicolumns(*[{**dict(dtype=0, x=at, u=at, rows=2, h=1, mc=3, how=ctypes.byref(how), c=at, stream=None), **a}[x]
                                                    for x in ("dtype", "x", "u", "rows", "h", "mc", "how", "c", "stream")])
    dist = lambda **a: lib.sbb_distill(*[{**dict(dtype=0, x=at, units=at, bytes=8, t=at, w=None, rows=2, h=1, mc=3, k=1, temp=1.0, loss=at, grad=at,
                                                    stream=None), **a}[x] for x in (
        "dtype", "x", "units", "bytes", "t", "w", "rows", "h", "mc", "k", "temp", "loss", "grad", "stream")])
    odd = ctypes.c_void_p(4098)
    for call, wrong in ((look, [dict(dtype=4), dict(dtype=-1), dict(bytes=2), dict(rows=-1), dict(l=-1), dict(n=0), dict(m=0), dict(w=None),
                                dict(c=None), dict(out=None), dict(w=odd), dict(c=odd)]),
                        (grad, [dict(dtype=4), dict(bytes=1), dict(rows=-1), dict(n=0), dict(out=None), dict(g=None), dict(c=None), dict(out=odd)]),
                        (draw, [dict(dtype=4), dict(rows=-1), dict(h=0), dict(mc=0), dict(how=None), dict(x=None), dict(u=None), dict(c=None),
                                dict(u=odd)]),
                        (dist, [dict(dtype=4), dict(bytes=3), dict(rows=-1), dict(h=0), dict(mc=0), dict(k=-1), dict(temp=0.0), dict(temp=-1.0),
                                dict(temp=math.inf), dict(x=None), dict(loss=None), dict(units=None), dict(t=None), dict(loss=odd)])):
        for a in wrong:
            assert call(**a) == _lib.ERR_INVALID, a
            assert lib.sbb_last_error()
    for call, wrong in ((look, [dict(rows=big), dict(l=big), dict(n=big), dict(m=big)]), (grad, [dict(rows=big), dict(l=big), dict(n=big)]),
                        (draw, [dict(rows=big), dict(h=big), dict(mc=big)]), (dist, [dict(rows=big), dict(mc=big), dict(k=big)])):
        for a in wrong:
            assert call(**a) == _lib.ERR_UNSUPPORTED, a
    if lib.sbb_device_count() == 0:
        assert look() == grad() == draw() == dist() == _lib.ERR_NO_DEVICE
    need = lib.sbb_lookup_gradient_workspace(0, 70000, 1, 50000, 64)
    assert need > 0
    for a in (dict(size=need - 1), dict(size=need, work=None), dict(size=need, work=ctypes.c_void_p(4104))):
        assert grad(rows=70000, l=1, n=50000, m=64, **a) == _lib.ERR_INVALID
