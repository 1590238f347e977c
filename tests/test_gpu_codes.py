"""Learned-code operators on the GPU -- embedding lookup, layer norm, counter-based dropout, their gradients -- against
their definitions in 64 bits.

Tolerances count roundings.  U = 2^-24 is half a step of fp32; half(t) = finfo(t).eps / 2 half a step of the output's type.
A sum of K fp32 terms in any order is off by at most (number of additions a term passes through) * U * sum |terms|; a row of C
values passes through at most 16 (register row) or C / 1024 + 8 (long row) additions in a lane and 10 between lanes:
`adds(C)`.
"""
import numpy as np
import pytest
import torch

from torch_nerf.amd import _lib, layers, ops, optim, synth
import torch_nerf.src.network as network
from torch_nerf.src.signal_encoder import PositionalEncoder

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF16, F16]
CODE = {F32: 0, BF16: 1, F16: 2}


def half(t):
    return torch.finfo(t).eps / 2


def step0(t):
    """What the subnormals add: half the smallest number (fp16's is not small)."""
    return 2.0 ** -25 if t == F16 else 1e-40


def adds(C):
    return 16 + 10 if C <= 16384 else C / 1024 + 18


def randn(g, *shape, t=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift).to(t).cuda()


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def close(got, want, tol, what=""):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = int((((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(1e30) * bad).reshape(-1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {i}: {got.reshape(-1)[i]} != "
                             f"{want.reshape(-1)[i]} (tolerance {tol.reshape(-1)[i]})")


# --------------------------------------------------------------------------- layer norm
def norm64(x, w, b, eps):
    """(y, mean, rstd, tolerance of y without its own rounding, of mean, of rstd)"""
    x = x.double()
    C = x.shape[-1]
    mu = x.mean(-1, keepdim=True)
    d = x - mu
    var = (d * d).mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    h = d * r
    t_mu = (adds(C) + 2) * U * x.abs().mean(-1, keepdim=True)
    # the variance: its sum, the rounding of each d, and the shift of the mean (second order in t_mu), then 1 / sqrt
    t_r = r * ((adds(C) / 2 + 5) * U + 0.5 * (t_mu * r) ** 2 + 0.5 * eps * U / (var + eps))
    t_y = w.abs() * (r * t_mu + d.abs() * t_r + 4 * U * h.abs()) + 2 * U * ((h * w).abs() + b.abs())
    return h * w + b, mu[..., 0], r[..., 0], t_y, t_mu[..., 0], t_r[..., 0]


def check_norm(x, w, b, eps=1e-5, what=""):
    y, mu, r = ops.layernorm(x, w, b, eps, want_stats=True)
    wy, wmu, wr, ty, tmu, tr = norm64(x, w, b, eps)
    assert y.dtype == x.dtype and mu.dtype == F32 and r.dtype == F32
    close(mu, wmu, tmu + U * wmu.abs(), what + " mean")
    close(r, wr, tr + 2 * U * wr.abs(), what + " rstd")
    close(y, wy, ty + half(x.dtype) * (wy.abs() + ty) + step0(x.dtype), what + " y")
    assert torch.equal(ops.layernorm(x, w, b, eps), y)
    return mu, r


def check_norm_backward(g, x, w, mu, r, M, what="", w_type=None):
    """Against the formula for the mean and rstd that it is given."""
    gx, gw, gb = ops.layernorm_backward(g, x, w, mu, r)
    C = x.shape[-1]
    xd, gd = x.double(), g.double()
    wd = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    rd = r.double()[..., None]
    h = (xd - mu.double()[..., None]) * rd
    q = gd * wd
    c0, c1 = q.mean(-1, keepdim=True), (q * h).mean(-1, keepdim=True)
    want = rd * (q - c0 - h * c1)
    k = adds(C)
    t = rd.abs() * U * ((k + 3) * q.abs().mean(-1, keepdim=True) + h.abs() * (k + 7) * (q * h).abs().mean(-1, keepdim=True)
                        + 4 * q.abs() + 3 * c0.abs() + 6 * (h * c1).abs())
    close(gx, want, t + half(x.dtype) * (want.abs() + t) + step0(x.dtype), what + " g_x")
    # a column: at most M additions in a lane, and 32 + 16 + 32 + 6 between lanes, wavefronts, slices and groups
    kc = M + 90
    dims = tuple(range(x.ndim - 1))
    for got, terms in ((gw, gd * h), (gb, gd)):
        s = terms.sum(dims)
        tt = (kc + 3) * U * terms.abs().sum(dims)
        assert got.dtype == (w.dtype if w is not None else x.dtype)
        close(got, s, tt + half(got.dtype) * (s.abs() + tt) + step0(got.dtype), what + " columns")


NORM_C = [1, 2, 3, 4, 5, 8, 16, 17, 31, 32, 33, 48, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025,
          2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384]


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("C", NORM_C)
def test_layernorm_rows(t, C):
    g = gen(C)
    for M in (1, 2, 67):
        x = randn(g, M, C, t=t, scale=1.5, shift=0.3)
        for wt in {t, F32}:
            w, b = randn(g, C, t=wt), randn(g, C, t=wt)
            mu, r = check_norm(x, w, b, what=f"{M}x{C} {t} {wt}")
            check_norm_backward(randn(g, M, C, t=t), x, w, mu, r, M, what=f"{M}x{C} {t} {wt}")
    mu, r = check_norm(x, None, None, what="plain")
    check_norm_backward(randn(g, M, C, t=t), x, None, mu, r, M, what="plain")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("C", [16385, 20011, 65536])
def test_layernorm_rows_beyond_a_workgroups_registers(t, C):
    g = gen(C)
    for M in (1, 3):
        x, w, b = randn(g, M, C, t=t, shift=-0.2), randn(g, C, t=t), randn(g, C, t=t)
        mu, r = check_norm(x, w, b, what=f"{M}x{C}")
        check_norm_backward(randn(g, M, C, t=t), x, w, mu, r, M, what=f"{M}x{C}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("M,C", [(5000, 7), (20011, 32), (9001, 256), (3001, 300), (2000, 1030), (1500, 4100),
                                 (9, 9000), (300, 9000), (1100, 5), (1025, 2), (4097, 3), (70, 512), (270000, 20), (262145, 130)])
def test_layernorm_many_rows(t, M, C):
    g = gen(M)
    x, w, b = randn(g, M, C, t=t), randn(g, C, t=t), randn(g, C, t=t)
    mu, r = check_norm(x, w, b, what=f"{M}x{C}")
    check_norm_backward(randn(g, M, C, t=t), x, w, mu, r, M, what=f"{M}x{C}")


def test_layernorm_shapes_and_strides():
    g = gen(1)
    wide = randn(g, 40, 300)
    w, b = randn(g, 100), randn(g, 100)
    x = wide[:, 101:201]                                   # columns of a matrix: read in place, odd offset
    assert not x.is_contiguous()
    y = ops.layernorm(x, w, b)
    assert y.is_contiguous() and torch.equal(y, ops.layernorm(x.contiguous(), w, b))
    mu, r = check_norm(x, w, b)
    go = randn(g, 40, 250)[:, 7:107]
    check_norm_backward(go, x, w, mu, r, 40)
    for xs in (wide[::2, 101:201], wide.t()[:100].t(), wide[:, :200:2]):
        assert torch.equal(ops.layernorm(xs, w, b), ops.layernorm(xs.contiguous(), w, b))
    x3 = randn(g, 3, 5, 100)
    y3, m3, r3 = ops.layernorm(x3, w, b, want_stats=True)
    assert y3.shape == (3, 5, 100) and m3.shape == (3, 5)
    assert torch.equal(y3.view(15, 100), ops.layernorm(x3.view(15, 100), w, b))
    assert torch.equal(ops.layernorm(x3.transpose(0, 1), w, b), y3.transpose(0, 1))
    one = randn(g, 100)
    y1, m1, r1 = ops.layernorm(one, w, b, want_stats=True)
    assert y1.shape == (100,) and m1.shape == ()
    g1 = ops.layernorm_backward(one, one, w, m1, r1)
    assert g1[0].shape == (100,)
    # a gradient that is one value for all (what .sum() hands back)
    full = torch.ones((), device="cuda").expand(40, 100)
    a, c = ops.layernorm_backward(full, x, w, mu, r), ops.layernorm_backward(full.contiguous(), x, w, mu, r)
    assert all(torch.equal(i, j) for i, j in zip(a, c))


@pytest.mark.parametrize("t", DTYPES)
def test_layernorm_empty_batches(t):
    w = torch.ones(33, device="cuda", dtype=t)
    x = torch.empty(0, 33, device="cuda", dtype=t)
    y, mu, r = ops.layernorm(x, w, w, want_stats=True)
    assert y.shape == (0, 33) and mu.shape == (0,)
    gx, gw, gb = ops.layernorm_backward(x, x, w, mu, r)
    assert gx.shape == (0, 33) and float(gw.abs().sum()) == 0.0 and float(gb.abs().sum()) == 0.0


def test_layernorm_keeps_digits_under_a_large_offset():
    """x = 1000 + noise: the variance about the mean; and rows of one value, whose deviation is exactly 0."""
    g = gen(2)
    x = (1000.0 + torch.randn(50, 256, generator=g)).cuda()
    check_norm(x, None, None)
    same = torch.full((4, 96), 3.5, device="cuda")
    y, mu, r = ops.layernorm(same, want_stats=True)
    assert torch.equal(y, torch.zeros_like(same)) and torch.equal(mu, same[:, 0])
    close(r, torch.full((4,), 1e-5).double().rsqrt(), torch.full((4,), 1e3 * U))


def check_norm_offset(x, w, b, eps=1e-5, what=""):
    """y, mean and rstd with bounds that an offset common to a row's values does not widen, but for the one rounding of a
    mean that is stored as fp32.

    Let k be the additions on a term's way.  The mean m that the deviations are summed about is off by delta: its own rounding
    U |mu|, and (k + 3) U mean|u| for a sum of numbers of the deviations' size, u = x - x0.  (Where m is less than 2^10
    deviations it may be the plain mean, off by 2^-9 of a deviation at most: 0.2 % of what follows, in bounds that count
    every rounding at its largest.)  d = x - m is off by U |d|, |d| <= D = |x - mu| + delta; e = mean(d) by (k + 3) U A, A = mean D.
    So the numerator x - m - e is off by U D + (k + 5) U A (the last two: the product e r).  The variance mean(d^2) - e^2 is
    off by (k + 6) U (V + delta^2) + 2 (delta + (k + 3) U A) (k + 3) U A + U delta^2, where V is the exact one; 1 / sqrt
    takes half of that relative to V + eps (0.75 with the higher orders, below 0.2) and 4 roundings."""
    y, mu, r = ops.layernorm(x, w, b, eps, want_stats=True)
    xd, C = x.double(), x.shape[-1]
    k = adds(C)
    m64 = xd.mean(-1, keepdim=True)
    dev = (xd - m64).abs()
    V = (dev * dev).mean(-1, keepdim=True)
    r64 = 1.0 / torch.sqrt(V + eps)
    delta = U * m64.abs() + (k + 3) * U * (xd - xd[..., :1]).abs().mean(-1, keepdim=True)
    D = dev + delta
    A = D.mean(-1, keepdim=True)
    t_e = (k + 3) * U * A
    t_V = ((k + 6) * U * (V + delta ** 2) + 2 * (delta + t_e) * t_e + U * delta ** 2) / (V + eps)
    assert float(t_V.max()) < 0.2, what
    t_r = r64 * (0.75 * t_V + 4 * U)
    h = (xd - m64) * r64
    wd, bd = w.double(), b.double()
    want = h * wd + bd
    t_y = wd.abs() * (r64 * (U * D + (k + 5) * U * A) + dev * t_r + 3 * U * h.abs()) + 2 * U * ((h * wd).abs() + bd.abs())
    close(mu, m64[..., 0], (t_e + 2 * U * (m64.abs() + delta))[..., 0], what + " mean")
    close(r, r64[..., 0], t_r[..., 0], what + " rstd")
    close(y, want, t_y + half(x.dtype) * (want.abs() + t_y) + step0(x.dtype), what + " y")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("C", [1, 3, 48, 255, 300, 600, 2047, 3000, 8191, 16000, 20011])
def test_layernorm_of_rows_with_an_offset(t, C):
    """Constant rows whose sums are inexact, and small deviations on a large offset (in 16 bits: what is left of them), in
    rows of one lane up to rows of several sweeps, few and many of them; and a first value far from all others."""
    g = gen(C)
    w, b = randn(g, C, t=t), randn(g, C, t=t)
    for M in (3, 1100 if C <= 4096 else 40):
        for offset, size in ((3333.3, 0.0), (1e4, 0.0), (-6e4, 0.0), (1e4, 0.01), (3e4, 1.0), (-777.7, 30.0)):
            x = randn(g, M, C, t=t, scale=size, shift=offset)
            check_norm_offset(x, w, b, what=f"{M}x{C} {t} {offset} {size}")
        x = randn(g, M, C, t=t)
        x[:, 0] = 1000.0
        check_norm_offset(x, w, b, what=f"{M}x{C} {t} first value")
    same = torch.full((5, C), 3333.3, device="cuda").to(t)
    y, mu, r = ops.layernorm(same, None, b, want_stats=True)
    assert torch.equal(y, b.expand(5, C)) and torch.equal(mu, same[:, 0].float())      # constant rows: 0 to the last bit


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("C", [2, 4, 9, 31, 64, 100, 128, 200, 256, 700, 3000, 20011])
def test_layernorm_rows_with_and_without_an_offset_side_by_side(t, C):
    """Rows that are summed once more and rows that are not, in one wavefront where the rows are short: every row has the bits
    that it has among rows of its own kind."""
    g = gen(C)
    M = 1200 if C <= 256 else 30
    x, w, b = randn(g, M, C, t=t), randn(g, C, t=t), randn(g, C, t=t)
    far = torch.rand(M, generator=g).cuda() < 0.5
    x[far] = (x[far].double() * 0.01 + 20000.0).to(t)
    x[::7] = 3333.3
    got = ops.layernorm(x, w, b, want_stats=True)
    kinds = (far & (torch.arange(M, device="cuda") % 7 != 0), ~far & (torch.arange(M, device="cuda") % 7 != 0),
             torch.arange(M, device="cuda") % 7 == 0)
    for rows in kinds:
        same = x[rows]
        many = same.repeat(-(-M // same.shape[0]), 1)[:M]          # as many rows: the same kernel
        want = ops.layernorm(many, w, b, want_stats=True)
        n = min(M, same.shape[0])
        assert all(torch.equal(a[rows], c[:n]) for a, c in zip(got, want))
    check_norm_offset(x, w, b, what=f"{C} {t}")


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("C", [3, 70, 3000, 20011])
def test_layernorm_of_the_lowest_value(t, C):
    """A row with its type's lowest value in it: the variance is beyond fp32, rstd 0 and the row its bias, as without an
    offset's care; rows beside it are untouched."""
    g = gen(C)
    x, b = randn(g, 4, C, t=t), randn(g, C, t=t)
    clean = ops.layernorm(x, None, b)
    x[1, 0] = x[2, C - 1] = torch.finfo(t).min
    y, mu, r = ops.layernorm(x, None, b, want_stats=True)
    assert bool((r[1:3] == 0).all()) and torch.equal(y[1:3], b.expand(2, C)) and bool(mu.isfinite().all())
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])


def odd(g, *shape, t=F32):
    """-3, -1, 1 or 3: products and sums of them are whole numbers, and none is 0."""
    return (2 * torch.randint(-1, 3, shape, generator=g) - 1).to(t).cuda()


# rows that every way of the backward pass takes: one workgroup, striding, the order of the addresses, several wavefronts a row
# (one and more rows a workgroup), longer than a workgroup's registers
WALKS = [(5, 3), (4097, 3), (3, 130), (9001, 20), (20011, 32), (262145, 130), (300000, 256), (70, 512), (5000, 600), (2000, 1030),
         (1500, 4100), (700, 9000), (1030, 16000), (130, 20011)]


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("M,C", WALKS)
def test_layernorm_column_sums_count_every_row_once(t, M, C):
    """The backward pass takes mean and rstd as they are given: with mean 0 and rstd 1 the weight's gradient is the sum of
    g x, the bias's that of g.  Of small odd numbers both are whole numbers below 9 M < 2^24, exact in fp32 in any order, and
    a row that is left out or counted twice changes every column."""
    assert 9 * M < 2 ** 24
    g = gen(M + C)
    x, go, w = odd(g, M, C, t=t), odd(g, M, C, t=t), torch.ones(C, device="cuda")
    gx, gw, gb = ops.layernorm_backward(go, x, w, torch.zeros(M, device="cuda"), torch.ones(M, device="cuda"))
    assert torch.equal(gw.double(), (go.double() * x.double()).sum(0)) and torch.equal(gb.double(), go.double().sum(0))
    few = ops.layernorm_backward(go, x, w.to(t), torch.zeros(M, device="cuda"), torch.ones(M, device="cuda"))
    assert torch.equal(few[1], gw.to(t)) and torch.equal(few[2], gb.to(t)) and torch.equal(few[0], gx)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("M,C", WALKS)
def test_layernorm_of_a_matrix_columns(t, M, C):
    """x and g as columns of wider matrices, of two widths, at odd offsets, and as every second row: the same bits as their
    copies give, forward and backward, in every kind of row."""
    g = gen(M + C)
    xs = torch.randn(M, C + 37, device="cuda").to(t)[:, 5:5 + C]
    gs = torch.randn(M, C + 12, device="cuda").to(t)[:, 3:3 + C]
    w, b = randn(g, C, t=t), randn(g, C, t=t)
    for x, go in ((xs, gs), (xs, gs.contiguous()), (xs[::2], gs[::2])):
        got = ops.layernorm(x, w, b, want_stats=True)
        want = ops.layernorm(x.contiguous(), w, b, want_stats=True)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        got = ops.layernorm_backward(go, x, w, *got[1:])
        want = ops.layernorm_backward(go.contiguous(), x.contiguous(), w, *want[1:])
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("M,C", [(9, 3), (9, 20), (9, 300), (9, 600), (9, 3000), (9, 9000), (9, 20011), (1100, 5), (1100, 130),
                                 (1100, 1030), (1100, 9000)])
def test_layernorm_infinities_and_nans_in_every_kind_of_row(t, M, C):
    """A value that is not finite, at the row's first, last or an inner place, makes its own row of y and of g_x NaN or
    infinite and no other; in g it reaches its column's sums, in x all of the weight's and none of the bias's."""
    g = gen(C)
    x, go, w, b = randn(g, M, C, t=t), randn(g, M, C, t=t), randn(g, C, t=t), randn(g, C, t=t)
    y0, mu0, r0 = ops.layernorm(x, w, b, want_stats=True)
    gx0, gw0, gb0 = ops.layernorm_backward(go, x, w, mu0, r0)
    xb = x.clone()
    xb[2, 0], xb[4, C - 1], xb[M - 2, C // 2] = float("inf"), float("nan"), -float("inf")
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[[2, 4, M - 2]] = True
    y, mu, r = ops.layernorm(xb, w, b, want_stats=True)
    assert torch.equal(y[~bad], y0[~bad]) and torch.equal(mu[~bad], mu0[~bad]) and torch.equal(r[~bad], r0[~bad])
    assert bool(y[bad].isnan().any(1).all()) and bool(r[bad].isnan().all()) and not bool(mu[bad].isfinite().any())
    gx, gw, gb = ops.layernorm_backward(go, xb, w, mu, r)
    assert torch.equal(gx[~bad], gx0[~bad]) and not bool(gx[bad].isfinite().any())
    assert bool(gw.isnan().all()) and torch.equal(gb, gb0)
    gbad = go.clone()
    gbad[3, C - 1] = float("inf")
    gx, gw, gb = ops.layernorm_backward(gbad, x, w, mu0, r0)
    rest = torch.arange(M, device="cuda") != 3
    assert torch.equal(gx[rest], gx0[rest]) and not bool(gx[3].isfinite().any())
    assert torch.equal(gb[:-1], gb0[:-1]) and not bool(gb[-1].isfinite()) and torch.equal(gw[:-1], gw0[:-1])
    assert not bool(gw[-1].isfinite())


def test_layernorm_infinities_and_nans_stay_in_their_rows():
    g = gen(3)
    x = randn(g, 9, 70)
    clean = ops.layernorm(x)
    x[2, 5], x[4, 69], x[7, 0] = float("inf"), float("nan"), -float("inf")
    y = ops.layernorm(x)
    bad = torch.tensor([2, 4, 7])
    good = torch.tensor([i for i in range(9) if i not in (2, 4, 7)])
    assert torch.equal(y[good], clean[good]) and bool(y[bad].isnan().any(1).all())


def test_layernorm_writes_only_its_rows():
    """Unaligned buffers in the middle of larger ones, through the C entries: what is around them stays."""
    lib, g = _lib.load(), gen(4)
    for t in DTYPES:
        for C in (5, 67, 1030):
            M = 6
            buf = torch.full((M * C + 40,), 7.0, device="cuda", dtype=t)
            x = randn(g, M * C + 3, t=t)[3:]
            size = x.element_size()
            rc = lib.nerf_layernorm(x.data_ptr(), C, CODE[t], M, C, None, None, 0, 1e-5, buf.data_ptr() + 19 * size, None,
                                    None, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert bool((buf[:19] == 7).all()) and bool((buf[19 + M * C:] == 7).all())
            assert torch.equal(buf[19:19 + M * C].view(M, C), ops.layernorm(x.view(M, C)))
            mu, r = ops.layernorm(x.view(M, C), want_stats=True)[1:]
            go = randn(g, M, C, t=t)
            gx = torch.full((M * C + 40,), 7.0, device="cuda", dtype=t)
            cols = torch.full((2, C + 10), 7.0, device="cuda")
            ws = torch.empty(lib.nerf_layernorm_backward_workspace_bytes(M, C, CODE[t]) + 16, dtype=torch.uint8, device="cuda")
            rc = lib.nerf_layernorm_backward(go.data_ptr(), C, x.data_ptr(), C, CODE[t], M, C, None, 0, mu.data_ptr(),
                                             r.data_ptr(), gx.data_ptr() + 21 * size, cols[0].data_ptr() + 20,
                                             cols[1].data_ptr() + 20, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert bool((gx[:21] == 7).all()) and bool((gx[21 + M * C:] == 7).all())
            assert bool((cols[:, :5] == 7).all()) and bool((cols[:, 5 + C:] == 7).all())


def test_layernorm_asks_only_for_what_is_wanted():
    g = gen(5)
    x, w, go = randn(g, 30, 48), randn(g, 48), randn(g, 30, 48)
    _, mu, r = ops.layernorm(x, w, want_stats=True)
    full = ops.layernorm_backward(go, x, w, mu, r)
    a = ops.layernorm_backward(go, x, w, mu, r, want_weight=False, want_bias=False)
    b = ops.layernorm_backward(go, x, w, mu, r, want_weight=False)
    c = ops.layernorm_backward(go, x, w, mu, r, want_bias=False)
    assert a[1] is None and a[2] is None and torch.equal(a[0], full[0])
    assert b[1] is None and torch.equal(b[2], full[2]) and c[2] is None and torch.equal(c[1], full[1])


def test_layernorm_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(8, device="cuda")
    s = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError):
        ops.layernorm(x.double())
    with pytest.raises(ValueError):
        ops.layernorm(x, w[:7])
    with pytest.raises(ValueError):
        ops.layernorm(x, w.half())
    with pytest.raises(ValueError):
        ops.layernorm(x.half(), w.bfloat16())
    with pytest.raises(ValueError):
        ops.layernorm(x.half(), w.half(), w)                # weight and bias of two types
    with pytest.raises(ValueError):
        ops.layernorm(x, w.cpu())
    with pytest.raises(ValueError):
        ops.layernorm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(RuntimeError, match="eps"):
        ops.layernorm(x, eps=-1.0)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x[:3], x, w, s, s)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x.half(), x, w, s, s)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x, x, w, s[:3], s)
    with pytest.raises(ValueError):
        ops.layernorm_backward(x, x, w, s.double(), s)


# --------------------------------------------------------------------------- embedding
EMB = [(1, 1, 1), (1, 5, 3), (7, 3, 16), (64, 10, 5), (300, 100, 48), (513, 1, 33), (1000, 4000, 64), (2000, 17, 257),
       (333, 70001, 12), (40, 300, 2049), (5, 9, 4100), (4097, 2, 8), (16384, 600, 20), (16385, 600, 20), (20000, 90000, 9),
       (70000, 37, 4),
       (1024, 50, 6), (1025, 50, 6), (32768, 3000, 7), (32769, 3000, 7), (3000, 40000, 1030), (50, 30000, 700),
       (40000, 100000, 264),
       (65536, 255, 33), (65537, 64, 33), (65537, 65, 12), (90000, 128, 6), (90000, 129, 6), (700, 255, 2100),
       (70000, 3000000, 2), (5000, 2000000, 3), (50000, 300, 1100), (300000, 1000, 5)]


def check_embedding_backward(go, ids, rows, scale, pad, what=""):
    got = ops.embedding_backward(go, ids, rows, scale, pad)
    n, dim = ids.numel(), go.shape[-1]
    gd, flat = go.double().reshape(n, dim), ids.reshape(-1).long()
    live = (flat >= 0) & (flat < rows)
    if pad is not None:
        live &= flat != pad
    flat, gd = flat[live].cpu(), gd[live].cpu()             # summed on the host, one after another
    want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, flat, gd)
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, flat, gd.abs())
    count = torch.bincount(flat, minlength=rows).double()[:, None]
    t = abs(scale) * U * (count + 3) * size
    want = want * float(np.float32(scale))
    assert got.dtype == go.dtype
    close(got, want, t + half(go.dtype) * (want.abs() + t) + step0(go.dtype) * (count > 0), what)
    assert torch.equal(got, ops.embedding_backward(go, ids, rows, scale, pad))      # the same bits again
    return got


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("n,rows,dim", EMB)
def test_embedding_and_its_gradient(t, n, rows, dim):
    g = gen(n + dim)
    table = randn(g, rows, dim, t=t)
    for kind, scale, pad, it in (("even", 1.0, None, torch.int64), ("skew", 3.7, 0, torch.int32), ("one", 0.5, None, torch.int64)):
        ids = torch.randint(rows, (n,), generator=g)
        if kind == "skew":
            ids = (ids.double() ** 3 / max(rows, 1) ** 2).long().clamp_(0, rows - 1)
        if kind == "one":
            ids[:] = rows - 1
        ids = ids.to(it).cuda()
        out = ops.embedding(table, ids, scale)
        want = table.double()[ids.long()] * float(np.float32(scale))
        tol = U * want.abs()
        close(out, want, tol + half(t) * (want.abs() + tol) + step0(t), kind)
        check_embedding_backward(randn(g, n, dim, t=t), ids, rows, scale, pad, what=f"{kind} {n} {rows} {dim} {t}")


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("n,rows,dim", [(786432, 100, 48), (786432, 1, 20), (786432, 255, 5), (300000, 1000, 33), (300000, 2000, 7),
                                        (32768, 300, 1100), (20000, 90000, 9), (1000, 4000, 600), (70000, 3, 1030)])
def test_embedding_gradient_counts_every_row_once(n, rows, dim, t):
    """Sums of small odd numbers are whole numbers below 3 n < 2^24, exact in fp32 in any order: what comes back is the exact
    sum, rounded once, and a row that is left out or counted twice changes every value of its id.  One id per run of 192
    (a ray's samples), ids that differ from sample to sample, and one id for all."""
    assert 3 * n < 2 ** 24
    g = gen(n + dim)
    go = odd(g, n, dim, t=t)
    rays = torch.randint(rows, ((n + 191) // 192,), generator=g).repeat_interleave(192)[:n]
    for ids in (rays, torch.randint(rows, (n,), generator=g), torch.full((n,), rows - 1)):
        got = ops.embedding_backward(go, ids.cuda(), rows)
        want = torch.zeros(rows, dim, dtype=torch.int32).index_add_(0, ids, go.to(torch.int32).cpu())
        assert torch.equal(got.cpu(), want.double().to(t))


def test_embedding_scale_one_is_a_copy():
    table = torch.randn(50, 37, device="cuda").half()
    ids = torch.randint(50, (4, 6), device="cuda")
    out = ops.embedding(table, ids)
    assert out.shape == (4, 6, 37) and torch.equal(out, table[ids])
    assert torch.equal(ops.embedding(table, ids[0, 0]), table[ids[0, 0]])           # one id without an axis
    wide = torch.randn(50, 80, device="cuda")
    assert torch.equal(ops.embedding(wide[:, 3:40], ids), wide[:, 3:40][ids])       # columns of a table, in place
    assert torch.equal(ops.embedding(wide.t(), ids.clamp(max=49)), wide.t()[ids.clamp(max=49)])


def test_embedding_ids_outside_the_table():
    table = torch.randn(10, 6, device="cuda")
    ids = torch.tensor([0, -1, 9, 10, 2 ** 40, -2 ** 63, 3], device="cuda")
    out = ops.embedding(table, ids)
    ok = torch.tensor([True, False, True, False, False, False, True], device="cuda")
    assert torch.equal(out[ok], table[ids[ok]]) and bool(out[~ok].isnan().all())
    check_embedding_backward(torch.randn(7, 6, device="cuda"), ids, 10, 2.0, None)
    check_embedding_backward(torch.randn(7, 6, device="cuda"), ids, 10, 2.0, 9)
    check_embedding_backward(torch.randn(7, 6, device="cuda"), torch.full((7,), -5, device="cuda"), 10, 1.0, None)
    big = torch.randint(-50, 300, (40000,), device="cuda")
    check_embedding_backward(torch.randn(40000, 6, device="cuda"), big, 200, 1.0, 7)


def test_embedding_infinities_and_nans_stay_in_their_rows():
    """A NaN in the gradient of a padded or unknown id is not read into any row; elsewhere it reaches its own row alone."""
    go = torch.randn(2000, 24, device="cuda")
    ids = torch.randint(1, 50, (2000,), device="cuda")
    ids[:300] = 0
    ids[300:310] = 77
    go[:310] = float("nan")
    got = ops.embedding_backward(go, ids, 50, 1.0, padding_idx=0)
    assert bool(got.isfinite().all()) and float(got[0].abs().sum()) == 0.0
    go[500, 3] = float("inf")
    row = int(ids[500])
    got2 = ops.embedding_backward(go, ids, 50, 1.0, padding_idx=0)
    assert got2[row, 3] == float("inf")
    got2[row, 3] = got[row, 3] = 0.0
    assert torch.equal(got2, got)


def test_embedding_empty_batches():
    table = torch.randn(10, 6, device="cuda")
    ids = torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops.embedding(table, ids).shape == (0, 6)
    g = ops.embedding_backward(torch.empty(0, 6, device="cuda"), ids, 10)
    assert g.shape == (10, 6) and float(g.abs().sum()) == 0.0


def test_embedding_writes_only_its_rows():
    lib = _lib.load()
    for t in DTYPES:
        for n, rows, dim in ((9, 5, 7), (300, 40, 35), (20000, 11, 3)):
            go = torch.randn(n, dim, device="cuda").to(t)
            ids = torch.randint(rows, (n,), device="cuda")
            buf = torch.full((rows * dim + 40,), 7.0, device="cuda", dtype=t)
            ws = torch.empty(lib.nerf_embedding_backward_workspace_bytes(n, rows, dim, CODE[t]) + 64, dtype=torch.uint8,
                             device="cuda")
            ws[-64:] = 77
            rc = lib.nerf_embedding_backward(go.data_ptr(), CODE[t], n, dim, ids.data_ptr(), 8, rows, 1.0, -1,
                                             buf.data_ptr() + 19 * buf.element_size(), ws.data_ptr(),
                                             torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and bool((ws[-64:] == 77).all())
            assert bool((buf[:19] == 7).all()) and bool((buf[19 + rows * dim:] == 7).all())
            assert torch.equal(buf[19:19 + rows * dim].view(rows, dim), ops.embedding_backward(go, ids, rows))
            out = torch.full((n * dim + 40,), 7.0, device="cuda", dtype=t)
            table = torch.randn(rows * dim + 1, device="cuda").to(t)[1:].view(rows, dim)
            rc = lib.nerf_embedding(table.data_ptr(), rows, dim, CODE[t], dim, ids.data_ptr(), 8, n, 1.0,
                                    out.data_ptr() + 19 * out.element_size(), torch.cuda.current_stream().cuda_stream)
            assert rc == 0 and bool((out[:19] == 7).all()) and bool((out[19 + n * dim:] == 7).all())
            assert torch.equal(out[19:19 + n * dim].view(n, dim), table[ids])


def test_embedding_offsets_beyond_32_bits():
    """A table of 2.2e9 values (4.4 GB in bf16): the last rows are looked up and written at their own places."""
    rows, dim = 1100003, 2048
    table = torch.zeros(rows, dim, device="cuda", dtype=BF16)
    table[-1], table[-2] = 3.0, 5.0
    ids = torch.tensor([rows - 1, 0, rows - 2], device="cuda")
    out = ops.embedding(table, ids)
    assert bool((out[0] == 3).all()) and bool((out[1] == 0).all()) and bool((out[2] == 5).all())
    del table
    g = ops.embedding_backward(out, ids, rows)
    assert bool((g[-1] == 3).all()) and bool((g[-2] == 5).all()) and int(torch.count_nonzero(g)) == 2 * dim


@pytest.mark.parametrize("n,seed", [(1, 0), (700, 1), (3000, 2), (40000, 3)])
def test_embedding_gradient_of_a_large_vocabulary(n, seed):
    """A table of 200 MB, whose rows are cleared in part before anything is known of the ids and in part by looking them up:
    rows of ids that occur hold their sums, every other row is exactly 0, whatever the memory held before."""
    rows, dim, g = 100003, 1030, gen(seed)
    for kind in ("even", "packed", "ends"):
        ids = torch.randint(rows, (n,), generator=g)
        if kind == "packed":                               # a run of neighbouring rows, each of them taken
            ids = (torch.arange(n) + 70001) % rows
        if kind == "ends":
            ids = torch.tensor([0, rows - 1, rows - 2, 1])[torch.randint(4, (n,), generator=g)]
        ids = ids.cuda()
        go = randn(g, n, dim, t=BF16)
        dirty = torch.full((rows, dim), float("nan"), device="cuda", dtype=BF16)
        del dirty                                          # the allocator hands the same memory out again
        got = ops.embedding_backward(go, ids, rows, 1.0)
        taken, back = torch.unique(ids, return_inverse=True)
        want = torch.zeros(taken.numel(), dim, dtype=torch.float64).index_add_(0, back.cpu(), go.double().cpu())
        size = torch.zeros(taken.numel(), dim, dtype=torch.float64).index_add_(0, back.cpu(), go.double().cpu().abs())
        t = U * (torch.bincount(back.cpu()).double()[:, None] + 3) * size
        close(got[taken], want, t + half(BF16) * (want.abs() + t), kind)
        got[taken] = 0
        assert int(torch.count_nonzero(got)) == 0 and bool(got.isfinite().all()), kind


@pytest.mark.parametrize("n,rows", [(10, 4000), (5000, 4000), (5000, 60), (50000, 4000)])
def test_embedding_gradient_without_a_single_known_id(n, rows):
    go = torch.randn(n, 300, device="cuda")
    for ids in (torch.full((n,), rows, device="cuda"), torch.full((n,), -1, device="cuda"), torch.full((n,), 7, device="cuda")):
        got = ops.embedding_backward(go, ids, rows, 1.0, padding_idx=7)
        assert int(torch.count_nonzero(got)) == 0 and bool(got.isfinite().all())


def test_embedding_refusals():
    table, ids = torch.zeros(10, 6, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    go = torch.zeros(4, 6, device="cuda")
    for bad in (lambda: ops.embedding(table.double(), ids), lambda: ops.embedding(table[0], ids),
                lambda: ops.embedding(table[:0], ids), lambda: ops.embedding(table, ids.float()),
                lambda: ops.embedding(table, ids.cpu()), lambda: ops.embedding(table, [0, 1]),
                lambda: ops.embedding_backward(go[:3], ids, 10), lambda: ops.embedding_backward(go, ids, 0),
                lambda: ops.embedding_backward(go, ids, 10, padding_idx=10),
                lambda: ops.embedding_backward(go, ids, 10, padding_idx=-1),
                lambda: ops.embedding_backward(go.double(), ids, 10)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="size out of range"):
        ops.embedding_backward(go, ids, 1 << 31)


# --------------------------------------------------------------------------- dropout
def kept(key, first, n, p):
    """The generator in numpy's unsigned 64-bit numbers."""
    with np.errstate(over="ignore"):
        e = np.arange(n, dtype=np.uint64) + np.uint64(first)
        z = (e >> np.uint64(1)) * np.uint64(0xD1342543DE82EF95) + np.uint64(key % 2 ** 64)
        z = synth._mix(z)
    bits = np.where(e % np.uint64(2) == 1, z >> np.uint64(32), z & np.uint64(0xFFFFFFFF))
    return torch.from_numpy(bits >= np.uint64(int(np.floor(p * 2.0 ** 32 + 0.5)))).cuda()


def check_dropout(x, p, key, first=0, residual=None):
    y = ops.dropout(x, p, key, first, residual)
    k = kept(key, first, x.numel(), p).view(x.shape)
    v = torch.where(k, x.double() / (1.0 - p) if p < 1 else 0.0, torch.zeros((), dtype=torch.float64, device="cuda"))
    t = 2 * U * v.abs()                                    # the scale's rounding and the product's
    want = v
    if residual is not None:
        want = v + residual.double()
        t = t + U * (want.abs() + t)
    close(y, want, t + half(x.dtype) * (want.abs() + t) + step0(x.dtype))
    if residual is None:
        assert bool((y[~k] == 0).all())
    return y


@pytest.mark.parametrize("t", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 8, 9, 63, 255, 1000, 4097, 100003])
def test_dropout_values_and_mask(t, n):
    g = gen(n)
    x, r = randn(g, n, t=t), randn(g, n, t=t)
    for p, key, first in ((0.1, 5, 0), (0.5, 2 ** 64 - 1, 1), (0.9, 0x123456789ABCDEF0, 2 ** 40 + 7), (0.0, 9, 3), (1.0, 9, 2),
                          (1e-12, 1, 0)):
        check_dropout(x, p, key, first)
        check_dropout(x, p, key, first, r)
    assert torch.equal(ops.dropout(x, 0.0, 1), x)
    assert torch.equal(ops.dropout(x, 1.0, 1), torch.zeros_like(x)) and torch.equal(ops.dropout(x, 1.0, 1, residual=r), r)


def test_dropout_of_a_shard_is_the_shard_of_the_dropout():
    x = torch.randn(9999, device="cuda")
    whole = ops.dropout(x, 0.3, 77, first=13)
    for lo, hi in ((0, 1), (1, 4), (1000, 5001), (5001, 9999)):
        assert torch.equal(ops.dropout(x[lo:hi].contiguous(), 0.3, 77, first=13 + lo), whole[lo:hi])
    y = ops.dropout(x[1:].view(2, 4999), 0.3, 77, first=14)                          # unaligned, another shape
    assert torch.equal(y.reshape(-1), whole[1:])
    xt = torch.randn(30, 50, device="cuda")
    assert torch.equal(ops.dropout(xt.t(), 0.3, 7), ops.dropout(xt.t().contiguous(), 0.3, 7))


def test_dropout_drops_what_it_drops():
    """An infinity or NaN in a dropped place gives 0; the share of dropped elements is p (6 sigma of the binomial)."""
    n, p = 1 << 20, 0.25
    x = torch.full((n,), float("nan"), device="cuda")
    y = ops.dropout(x, p, 3)
    k = kept(3, 0, n, p)
    assert bool((y[~k] == 0).all()) and bool(y[k].isnan().all())
    assert abs(int(k.sum()) - n * (1 - p)) <= 6 * (n * p * (1 - p)) ** 0.5
    other = kept(4, 0, n, p)                                # keys give masks of their own
    assert abs(int((k & other).sum()) - n * (1 - p) ** 2) <= 6 * (n * (1 - p) ** 2 * (1 - (1 - p) ** 2)) ** 0.5


def test_dropout_of_more_elements_than_32_bits_count():
    """2^31 + 100 elements (4.3 GB): more than one launch takes; pieces around the seam and the end against smaller calls."""
    n = 2 ** 31 + 100
    x = torch.ones(n, device="cuda", dtype=BF16)
    y = ops.dropout(x, 0.25, 9, first=3)
    for lo, hi in ((0, 5000), (2 ** 31 - 5001, 2 ** 31 + 77), (n - 100, n)):
        assert torch.equal(y[lo:hi], ops.dropout(x[lo:hi].clone(), 0.25, 9, first=3 + lo))
    kept_share = float((y != 0).double().mean())
    assert abs(kept_share - 0.75) <= 6 * (0.75 * 0.25 / n) ** 0.5


def test_dropout_key_tensor():
    x = torch.randn(777, device="cuda")
    for key in (0, 5, 2 ** 63 + 11, 2 ** 64 - 3):
        kt = torch.tensor([key - 2 ** 64 if key >= 2 ** 63 else key], device="cuda")
        assert torch.equal(ops.dropout(x, 0.4, kt), ops.dropout(x, 0.4, key))
    assert torch.equal(ops.dropout(x, 0.4, -3), ops.dropout(x, 0.4, 2 ** 64 - 3))


def test_dropout_refusals():
    x = torch.zeros(8, device="cuda")
    for bad in (lambda: ops.dropout(x, -0.1, 1), lambda: ops.dropout(x, 1.1, 1), lambda: ops.dropout(x, float("nan"), 1),
                lambda: ops.dropout(x, 0.5, 1, first=-1), lambda: ops.dropout(x, 0.5, 1, first=2 ** 63 - 8),
                lambda: ops.dropout(x.double(), 0.5, 1), lambda: ops.dropout(x, 0.5, 1, residual=x[:7]),
                lambda: ops.dropout(x, 0.5, 1, residual=x.half()), lambda: ops.dropout(x, 0.5, torch.zeros(2, device="cuda").long()),
                lambda: ops.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------------------- gradients through autograd
def stage64(table, ids, w, b, p, key, scale, eps=1e-5):
    """embedding -> layer norm -> dropout in 64 bits."""
    e = table[ids] * scale
    mu = e.mean(-1, keepdim=True)
    d = e - mu
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w + b
    k = kept(key, 0, y.numel(), p).view(y.shape)
    return torch.where(k, y / (1 - p), torch.zeros((), dtype=torch.float64, device="cuda"))


def test_gradients_against_formula_and_differences():
    """The three operators in a row in fp32, their gradients against autograd of the 64-bit formula and against central
    differences of it.  Tolerances: every value passes fewer than 60 roundings along the chain (16 + 10 additions twice in
    the norm, products, one per repetition of an id), each at most U of the sum of the magnitudes it is made of; the
    magnitudes of this case keep that below 400 U of the largest gradient."""
    g = gen(8)
    rows, dim, n, p, key, scale = 6, 20, 40, 0.25, 99, 1.5
    table, w, b = (randn(g, rows, dim), randn(g, dim), randn(g, dim))
    ids = torch.randint(rows, (n,), generator=g).cuda()
    up = randn(g, n, dim)
    leaves = [t.clone().requires_grad_(True) for t in (table, w, b)]
    e = ops.EmbeddingFunction.apply(leaves[0], ids, scale, None)
    y = ops.LayerNormFunction.apply(e, leaves[1], leaves[2], 1e-5)
    out = ops.DropoutFunction.apply(y, p, key)
    got = torch.autograd.grad(out, leaves, up)
    lead = [t.double().requires_grad_(True) for t in (table, w, b)]
    ref = stage64(*lead[:1], ids, *lead[1:], p, key, scale)
    want = torch.autograd.grad(ref, lead, up.double())
    close(out.detach(), ref.detach(), 400 * U * ref.detach().abs().max().expand_as(ref))
    for a, c in zip(got, want):
        close(a, c, (400 * U * c.abs().max()).expand_as(c))
    step = 1e-5
    for k in range(3):
        v = torch.randn(lead[k].shape, generator=g, dtype=torch.float64).cuda()
        args = [t.detach() for t in lead]

        def f(s):
            moved = [t + s * v if i == k else t for i, t in enumerate(args)]
            return float((stage64(moved[0], ids, moved[1], moved[2], p, key, scale) * up.double()).sum())
        slope = (f(step) - f(-step)) / (2 * step)
        mine = float((got[k].double() * v).sum())
        # differences: third derivatives of order 10^3 at this size, times step^2; the gradient: as above, summed over v
        assert abs(slope - mine) <= 1e-6 + 400 * U * float(got[k].abs().max()) * float(v.abs().sum()), (k, slope, mine)


def test_functions_give_gradients_only_where_asked():
    g = gen(9)
    x, w, b, r = randn(g, 5, 12), randn(g, 12), randn(g, 12), randn(g, 5, 12)
    for need in range(8):
        ts = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b))]
        y = ops.LayerNormFunction.apply(*ts, 1e-5)
        assert y.requires_grad == bool(need)
        if need:
            y.sum().backward()
        assert [t.grad is not None for t in ts] == [bool(need >> i & 1) for i in range(3)]
    for t in DTYPES:                                        # 16-bit rows with fp32 weights, with a bias alone
        xt = x.detach().clone().to(t).requires_grad_(True)
        bt = b.clone().requires_grad_(True)
        ops.LayerNormFunction.apply(xt, None, bt, 1e-5).sum().backward()
        assert xt.grad.dtype == t and bt.grad.dtype == F32 and bool((bt.grad == 5).all())
    xr, rr = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
    ops.DropoutFunction.apply(xr, 0.5, 3, 0, rr).backward(r)
    assert torch.equal(rr.grad, r) and torch.equal(xr.grad, ops.dropout(r, 0.5, 3))
    kt = torch.tensor([3], device="cuda")
    xk = x.clone().requires_grad_(True)
    y = ops.DropoutFunction.apply(xk, 0.5, kt)
    y.backward(r, retain_graph=True)
    assert torch.equal(xk.grad, xr.grad)
    kt += 1                                                 # the key may not change between the passes
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(r)
    shared = x.clone().requires_grad_(True)                 # one input as value and residual
    ops.DropoutFunction.apply(shared, 0.5, 3, 0, shared).backward(r)
    assert torch.equal(shared.grad, r + ops.dropout(r, 0.5, 3))


def test_layernorm_bias_alone_keeps_its_digits():
    """16-bit rows with an fp32 bias and no weight: the bias's gradient is an fp32 sum (99 additions at most along a term's
    way, below 100 U of the magnitudes), not one that was rounded to 16 bits first."""
    g = gen(21)
    for t in (BF16, F16):
        x, b, up = randn(g, 99, 40, t=t), randn(g, 40), randn(g, 99, 40, t=t)
        bias = b.clone().requires_grad_(True)
        ops.LayerNormFunction.apply(x, None, bias, 1e-5).backward(up)
        close(bias.grad, up.double().sum(0), 100 * U * up.double().abs().sum(0))
        mu, r = ops.layernorm(x, None, b, want_stats=True)[1:]
        assert ops.layernorm_backward(up, x, None, mu, r)[2].dtype == t
        w = randn(g, 40, t=t)
        with pytest.raises(ValueError, match="bias_dtype"):
            ops.layernorm_backward(up, x, w, mu, r, bias_dtype=F32)
        with pytest.raises(ValueError, match="bias_dtype"):
            ops.layernorm_backward(up, x, None, mu, r, bias_dtype=torch.float64)


def test_modules_in_a_conditioned_network():
    """A code per view, normalised and dropped out, behind NeRF's view direction, trained with the network under FusedAdam:
    forward and all gradients against torch in 64 bits, and the whole step without a host synchronisation in between."""
    torch.manual_seed(3)
    views, width, M = 11, 16, 640
    codes = layers.Embedding(views, width, scale=0.5).cuda()
    norm = layers.LayerNorm(width).cuda()
    drop = layers.Dropout(0.25, seed=4)
    net = network.NeRF(63, 27 + width).cuda()
    ids = torch.randint(views, (M // 64,), device="cuda").repeat_interleave(64)
    pe, de = PositionalEncoder(3, 10, True), PositionalEncoder(3, 4, True)
    pos, vd = pe.encode(torch.randn(M, 3, device="cuda")), de.encode(torch.randn(M, 3, device="cuda"))
    g_s, g_c = torch.randn(M, device="cuda"), torch.randn(M, 3, device="cuda")
    code = drop(norm(codes(ids)))
    code.retain_grad()
    sigma, rgb = net(pos, torch.cat([vd, code], 1))
    ((sigma * g_s).sum() + (rgb * g_c).sum()).backward()
    key = layers._mix_int((4 * 0x9E3779B97F4A7C15 + 0) ^ 0xD6E8FEB86659FD93)
    t64, w64, b64 = (t.detach().double().requires_grad_(True) for t in (codes.weight, norm.weight, norm.bias))
    ref = stage64(t64, ids, w64, b64, 0.25, key, 0.5)
    close(code.detach(), ref.detach(), 400 * U * ref.detach().abs().max().expand_as(ref))
    want = torch.autograd.grad(ref, (t64, w64, b64), code.grad.double())
    for p, c in zip((codes.weight, norm.weight, norm.bias), want):
        # as above, and an id repeats up to M times: its sum passes M additions
        size = code.grad.double().abs().sum() / views
        close(p.grad, c, ((400 * float(c.abs().max()) + M * float(size)) * U * torch.ones_like(c)))
    opt = optim.FusedAdam([*codes.parameters(), *norm.parameters(), *net.parameters()], lr=1e-3)
    before = codes.weight.detach().clone()
    opt.step()
    used = torch.zeros(views, dtype=torch.bool, device="cuda")
    used[ids] = True
    assert torch.equal((codes.weight.detach() != before).any(1), used & (codes.weight.grad != 0).any(1))
    assert drop.calls == 1 and not torch.equal(drop(code), drop(code))
    drop.eval()
    assert drop(code) is code


def test_default_dropout_modules_draw_masks_of_their_own():
    """Share of elements that two modules both keep on their n-th call: (1 - p)^2 within 6 sigma, not 1 - p."""
    n, p = 1 << 18, 0.5
    x = torch.ones(n, device="cuda")
    a, b = layers.Dropout(p), layers.Dropout(p)
    for _ in range(3):
        both = int(((a(x) != 0) & (b(x) != 0)).sum())
        assert abs(both - n / 4) <= 6 * (n * 0.25 * 0.75) ** 0.5
    same = layers.Dropout(p, seed=a.seed)
    a.calls = 0
    assert torch.equal(a(x), same(x))


# --------------------------------------------------------------------------- streams and graphs
def test_on_another_stream_and_two_at_once():
    g = gen(10)
    x, w, go = randn(g, 3000, 256), randn(g, 256), randn(g, 3000, 256)
    ids = torch.randint(40, (3000,), generator=g).cuda()

    def all_of_it():
        y, mu, r = ops.layernorm(x, w, None, want_stats=True)
        return [y, *ops.layernorm_backward(go, x, w, mu, r), ops.embedding_backward(go, ids, 40),
                ops.embedding(w.view(16, 16), ids % 16, 2.0), ops.dropout(x, 0.3, 5)]
    want = all_of_it()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(all_of_it())
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_captured_and_replayed():
    """Forward and backward of all three in one graph, two graphs of different sizes in turn, new inputs and keys between
    the replays, every replay against the eager result."""
    graphs = []
    for n, rows, dim in ((900, 30, 64), (17000, 500, 20)):
        st = {"ids": torch.randint(rows, (n,), device="cuda"), "table": torch.randn(rows, dim, device="cuda"),
              "w": torch.randn(dim, device="cuda"), "g": torch.randn(n, dim, device="cuda"),
              "key": torch.tensor([1], device="cuda"), "rows": rows}

        def step(st=st):
            e = ops.embedding(st["table"], st["ids"], 1.25)
            y, mu, r = ops.layernorm(e, st["w"], None, want_stats=True)
            out = ops.dropout(y, 0.2, st["key"])
            gy = ops.dropout_backward(st["g"], 0.2, st["key"])
            ge, gw, gb = ops.layernorm_backward(gy, e, st["w"], mu, r)
            return out, ge, gw, gb, ops.embedding_backward(ge, st["ids"], st["rows"], 1.25, 3)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        graphs.append((graph, st, step, res))
    for turn in range(4):
        for graph, st, step, res in graphs:
            st["ids"].copy_(torch.randint(st["rows"], st["ids"].shape, device="cuda"))
            st["g"].normal_()
            st["key"] += 1
        for graph, _, _, _ in graphs:
            graph.replay()
        for _, _, step, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(step(), res))
        torch.cuda.synchronize()


def test_modules_captured_with_their_backward_pass():
    """The modules' forward and autograd's backward pass in one graph (no eager graph of the parameters lives meanwhile),
    replayed with new inputs and keys, every replay against the eager result."""
    torch.manual_seed(22)
    codes, norm = layers.Embedding(50, 24, scale=0.5, padding_idx=0).cuda(), layers.LayerNorm(24).cuda()
    drop = layers.Dropout(0.3)
    params = [*codes.parameters(), *norm.parameters()]
    ids, up = torch.randint(50, (5000,), device="cuda"), torch.randn(5000, 24, device="cuda")
    key = torch.tensor([7], device="cuda")

    def step():
        out = drop(norm(codes(ids)), key=key)
        return [out.detach(), *torch.autograd.grad(out, params, up)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for turn in range(4):
        ids.copy_(torch.randint(50, ids.shape, device="cuda"))
        up.normal_()
        key += 1
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, res))


def test_dropout_module_refuses_a_capture_without_a_key():
    drop = layers.Dropout(0.5)
    x = torch.randn(64, device="cuda")
    key = torch.tensor([3], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="key tensor"):
            drop(x)
        y = drop(x, key=key)
    graph.replay()
    assert torch.equal(y, ops.dropout(x, 0.5, 3))


@pytest.mark.parametrize("n,dim", [(786432, 48), (16384, 1024)])
def test_large_batches(n, dim):
    """The sizes of a training batch: all samples of 4096 rays with the code of one view each, and one view for all."""
    t = F32 if dim == 48 else BF16
    go = torch.randn(n, dim, device="cuda").to(t)
    ids = torch.randint(100, (n // 64,), device="cuda").repeat_interleave(64)
    check_embedding_backward(go, ids, 100, 1.0, None, "rays")
    check_embedding_backward(go, torch.full((n,), 3, device="cuda"), 5, 1.0, None, "one view")
    check_embedding_backward(go, torch.randint(131072, (n,), device="cuda"), 131072, 2.0, 1, "many rows")
