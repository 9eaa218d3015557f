"""Dense operators (similaripy_amd.dense, include/sp_dense.h) against their formulas in 64 bits.

Bounds.  u = 2^-24 is half a step of float32, h half a step of the result's type.  A float32 sum of m products, in whatever order, is
off by at most (m + 1) u times the sum of the terms' magnitudes; the result is then rounded once (h times its value, and half the
smallest subnormal of float16).  What the exponentials add is derived where it is used.
"""
from __future__ import annotations

import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from similaripy_amd import _abi, dense

ROOT = Path(__file__).resolve().parent.parent
HEADER = (ROOT / "include" / "sp_dense.h").read_text()
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150


def check(got, want, bound, what=""):
    """|got - want| <= bound elementwise, the same infinities, the same NaNs."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want) if not torch.is_tensor(bound) else bound.double().cpu().expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    d = (got[fin] - want[fin]).abs()
    worst = (d - bound[fin]).max().item() if d.numel() else -1.0
    assert worst <= 0, f"{what}: off by {d.max().item():.3e}, {worst:.3e} over the bound"


def csr(rng, n, vocab, mean, dtype=torch.int32, empty=0.2, bad=0.0):
    """Row pointers and ids: ragged rows, some empty, ids repeat, a share `bad` outside the vocabulary."""
    lens = rng.poisson(mean, n)
    lens[rng.random(n) < empty] = 0
    indptr = np.zeros(n + 1, np.int64)
    np.cumsum(lens, out=indptr[1:])
    ids = rng.integers(0, max(1, vocab), indptr[-1])
    if bad:
        ids = np.where(rng.random(ids.shape[0]) < bad, rng.choice([-1, -7, vocab, vocab + 3], ids.shape[0]), ids)
    return torch.from_numpy(indptr).to(dtype), torch.from_numpy(ids).to(dtype)


# ---- embedding rows ------------------------------------------------------------------------------------------------------------

def embed_ref(table, ids, indptr, data, scale):
    """(result, sum of magnitudes, longest row) in 64 bits."""
    t, ids = table.double().cpu(), ids.reshape(-1).long().cpu()
    n = ids.numel() if indptr is None else indptr.numel() - 1
    row = torch.arange(n) if indptr is None else torch.repeat_interleave(torch.arange(n), (indptr[1:] - indptr[:-1]).long().cpu())
    w = torch.ones(ids.numel(), dtype=torch.float64) if data is None else data.double().cpu()
    ok = (ids >= 0) & (ids < t.shape[0])
    terms = t[ids[ok]] * w[ok][:, None] * scale
    out, mag = torch.zeros(n, t.shape[1], dtype=torch.float64), torch.zeros(n, t.shape[1], dtype=torch.float64)
    out.index_add_(0, row[ok], terms)
    mag.index_add_(0, row[ok], terms.abs())
    longest = int(torch.bincount(row, minlength=max(1, n)).max()) if row.numel() else 0
    return out, mag, longest


def embed_grad_ref(grad, ids, n_vocab, indptr, data, scale):
    g, ids = grad.double().cpu(), ids.reshape(-1).long().cpu()
    n = ids.numel() if indptr is None else indptr.numel() - 1
    row = torch.arange(n) if indptr is None else torch.repeat_interleave(torch.arange(n), (indptr[1:] - indptr[:-1]).long().cpu())
    w = torch.ones(ids.numel(), dtype=torch.float64) if data is None else data.double().cpu()
    ok = (ids >= 0) & (ids < n_vocab)
    terms = g[row[ok]] * w[ok][:, None] * scale
    out, mag = torch.zeros(n_vocab, g.shape[1], dtype=torch.float64), torch.zeros(n_vocab, g.shape[1], dtype=torch.float64)
    out.index_add_(0, ids[ok], terms)
    mag.index_add_(0, ids[ok], terms.abs())
    longest = int(torch.bincount(ids[ok], minlength=1).max()) if ids[ok].numel() else 0
    return out, mag, longest


def sum_bound(out, mag, m, dtype):
    # m products and additions, the weight's product and the scale: (m + 3) u of the magnitudes; one rounding of the result
    return (m + 3) * U * mag + half_step(dtype) * (out.abs() + (m + 3) * U * mag) + tiny(dtype)


EMBED_DIMS = [1, 3, 8, 64, 129, 512, 1000]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", EMBED_DIMS)
def test_embed_lookup(dtype, dim):
    rng = np.random.default_rng(dim)
    table = torch.from_numpy(rng.standard_normal((57, dim))).to(dtype).cuda()
    for n, it in ((1, torch.int64), (5, torch.int32), (1031, torch.int64)):
        ids = torch.from_numpy(rng.integers(-3, 60, n)).to(it).cuda()
        got = dense.embed_rows(table, ids, scale=1.7)
        want, mag, m = embed_ref(table, ids, None, None, 1.7)
        check(got, want, sum_bound(want, mag, 1, dtype), f"n={n}")
        assert got.dtype == dtype


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", EMBED_DIMS)
@pytest.mark.parametrize("weighted", [False, True])
def test_embed_bags(dtype, dim, weighted):
    rng = np.random.default_rng(100 + dim)
    for n, vocab, mean, it in ((1, 9, 3, torch.int32), (67, 211, 11, torch.int64), (203, 97, 70, torch.int32)):
        table = torch.from_numpy(rng.standard_normal((vocab, dim))).to(dtype).cuda()
        indptr, ids = csr(rng, n, vocab, mean, it, bad=0.1)
        data = torch.from_numpy(rng.standard_normal(ids.numel()).astype(np.float32)).cuda() if weighted else None
        got = dense.embed_rows(table, ids.cuda(), indptr.cuda(), data, scale=0.5)
        want, mag, m = embed_ref(table, ids, indptr, data, 0.5)
        check(got, want, sum_bound(want, mag, m, dtype), f"n={n}")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_layouts(dtype):
    """Padded rows, a table that starts off 16 bytes, indices of two dimensions, a caller's output with padded rows, no rows at all."""
    rng = np.random.default_rng(5)
    big = torch.from_numpy(rng.standard_normal((40, 75))).to(dtype).cuda()
    table = big[3:, 1:68]
    ids = torch.from_numpy(rng.integers(0, 37, (4, 9))).cuda()
    want, mag, _ = embed_ref(table, ids, None, None, 1.0)
    got = dense.embed_rows(table, ids)
    assert got.shape == (4, 9, 67)
    check(got.reshape(36, 67), want, sum_bound(want, mag, 1, dtype))
    store = torch.full((36, 80), 7.0, dtype=dtype, device="cuda")
    res = dense.embed_rows(table, ids.reshape(-1), out=store[:, 5:72])
    assert res.data_ptr() == store[:, 5:72].data_ptr()
    check(store[:, 5:72], want, sum_bound(want, mag, 1, dtype))
    assert (store[:, :5] == 7).all() and (store[:, 72:] == 7).all()
    assert dense.embed_rows(table, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 67)
    assert (dense.embed_rows(table[:0], ids) == 0).all()                         # an empty vocabulary: every id is outside
    none = dense.embed_rows(table, torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert none.shape == (3, 67) and (none == 0).all()


@gpu
def test_embed_rows_outside_indptr_are_not_read():
    """Row pointers that leave [0, nnz] are cut to it."""
    table = torch.ones(4, 8, device="cuda")
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    indptr = torch.tensor([-2, 3, 3, 900], dtype=torch.int32, device="cuda")
    assert dense.embed_rows(table, ids, indptr)[:, 0].tolist() == [3.0, 0.0, 2.0]
    g = dense.embed_rows_grad(torch.tensor([[1.0], [10.0], [100.0]], device="cuda").repeat(1, 8), ids, 4, indptr)
    assert g[0, 0].item() == 203.0 and (g[1:] == 0).all()
    nobody = torch.zeros(1, dtype=torch.int32, device="cuda")                    # no rows at all, though there are entries
    assert (dense.embed_rows_grad(torch.ones(0, 8, device="cuda"), ids, 4, nobody) == 0).all() and dense.embed_rows(table, ids, nobody).shape == (0, 8)
    indptr = torch.tensor([2, 4], dtype=torch.int32, device="cuda")              # entries before the first row and behind the last belong to none
    assert dense.embed_rows(table, ids, indptr)[0, 0].item() == 2.0
    assert dense.embed_rows_grad(torch.ones(1, 8, device="cuda"), ids, 4, indptr)[0, 0].item() == 2.0


GRADS = [  # n, vocab, mean entries of a row (0: lookup), share of bad ids
    (1, 1, 0, 0.0), (1, 700, 0, 0.0), (2, 3, 0, 0.5), (777, 50, 0, 0.05), (5000, 3, 0, 0.0), (9001, 70_000, 0, 0.01),
    (1024, 90_000, 0, 0.1), (1025, 5000, 0, 0.1), (1000, 5, 0, 0.2), (8192, 2000, 0, 0.0), (8193, 2000, 0, 0.0), (60, 3000, 15, 0.1),
    (1, 40, 5, 0.0), (300, 511, 30, 0.1), (300, 512, 30, 0.1), (64, 300_000, 20, 0.0), (900, 7, 60, 0.0),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,mean,bad", GRADS)
@pytest.mark.parametrize("dim", [1, 24, 129])
def test_embed_grad(dtype, n, vocab, mean, bad, dim):
    rng = np.random.default_rng(n + vocab + dim)
    grad = torch.from_numpy(rng.standard_normal((n, dim))).to(dtype).cuda()
    it = torch.int32 if (n + dim) % 2 else torch.int64
    if mean:
        indptr, ids = csr(rng, n, vocab, mean, it, bad=bad)
        data = torch.from_numpy(rng.standard_normal(ids.numel()).astype(np.float32)).cuda() if dim != 24 else None
        indptr = indptr.cuda()
    else:
        ids = rng.integers(0, vocab, n)
        ids = torch.from_numpy(np.where(rng.random(n) < bad, -1, ids)).to(it)
        indptr = data = None
    want, mag, m = embed_grad_ref(grad, ids, vocab, indptr, data, 3.0)
    for out_dtype in {dtype, torch.float32}:
        got = dense.embed_rows_grad(grad, ids.cuda(), vocab, indptr, data, scale=3.0, dtype=out_dtype)
        assert got.dtype == out_dtype
        check(got, want, sum_bound(want, mag, m, out_dtype), str(out_dtype))
        again = dense.embed_rows_grad(grad, ids.cuda(), vocab, indptr, data, scale=3.0, dtype=out_dtype)
        assert torch.equal(got, again)


@gpu
@pytest.mark.parametrize("dim", [64, 700])
def test_embed_grad_one_popular_id(dim):
    """Nearly all of many entries name one id: its run spans most chunks of the sorted entries."""
    rng = np.random.default_rng(1)
    n, vocab = 300_000 if dim == 64 else 40_000, 1000
    ids = np.where(rng.random(n) < 0.9, 317, rng.integers(0, vocab, n))
    grad = torch.from_numpy(rng.standard_normal((n, dim)).astype(np.float32)).cuda()
    got = dense.embed_rows_grad(grad, torch.from_numpy(ids).cuda(), vocab)
    want, mag, m = embed_grad_ref(grad, torch.from_numpy(ids), vocab, None, None, 1.0)
    # sums of chunks, joined: additions in sequence are at most a chunk's and the chunks', far fewer than m; m holds all the same
    check(got, want, sum_bound(want, mag, m, torch.float32))
    # (the bound above is loose for the popular id: a dropped or doubled entry would move its sum by about one)
    assert (got[317].double().cpu() - want[317]).abs().max() < 0.05


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_embed_grad_accumulate_and_layouts(dtype):
    rng = np.random.default_rng(9)
    vocab, dim = 301, 70
    ids = torch.from_numpy(rng.integers(0, 60, 500)).cuda()
    store = torch.from_numpy(rng.standard_normal((500, 90))).to(dtype).cuda()
    grad = store[:, 3:73]
    base = torch.from_numpy(rng.standard_normal((vocab, 77))).to(dtype).cuda()
    out = base.clone()
    res = dense.embed_rows_grad(grad, ids, vocab, out=out[:, 2:72], accumulate=True)
    assert res.data_ptr() == out[:, 2:72].data_ptr()
    want, mag, m = embed_grad_ref(grad, ids, vocab, None, None, 1.0)
    full = want + base[:, 2:72].double().cpu()
    check(out[:, 2:72], full, sum_bound(full, mag + base[:, 2:72].double().cpu().abs(), m + 1, dtype))
    assert torch.equal(out[60:], base[60:])                                       # ids that do not occur: not touched
    assert torch.equal(out[:, :2], base[:, :2]) and torch.equal(out[:, 72:], base[:, 72:])
    out = torch.full((vocab, 77), 5.0, dtype=dtype, device="cuda")                # without: every row is written, nothing beside it
    dense.embed_rows_grad(grad, ids, vocab, out=out[:, 2:72])
    check(out[:, 2:72], want, sum_bound(want, mag, m, dtype))
    assert (out[:, :2] == 5).all() and (out[:, 72:] == 5).all()
    none = dense.embed_rows_grad(grad[:0], ids[:0], vocab)
    assert none.shape == (vocab, dim) and (none == 0).all()
    assert torch.equal(dense.embed_rows_grad(torch.ones(1, dim, device="cuda", dtype=dtype).expand(500, dim), ids, vocab),
                       dense.embed_rows_grad(torch.ones(500, dim, device="cuda", dtype=dtype), ids, vocab))     # a broadcast gradient


@gpu
@pytest.mark.parametrize("dtype,rows,dim", [(torch.float32, 2200, 512), (torch.bfloat16, 2300, 1024), (torch.float16, 1100, 2048), (torch.float32, 1100, 1024),
                                            (torch.float32, 3000, 384), (torch.float32, 1500, 768), (torch.bfloat16, 900, 4096)])
def test_embed_grad_wide_rows(dtype, rows, dim):
    """Rows beyond the L2 of an XCD, cut by columns where they can be; short runs, runs over a few chunks of the sorted entries and over many."""
    rng = np.random.default_rng(dim + rows)
    n, vocab = rows * 17, 70
    ids = np.concatenate([rng.integers(0, vocab, n // 2), np.minimum(rng.zipf(1.3, n - n // 2) - 1, vocab)])      # the id `vocab` is outside
    ids = torch.from_numpy(rng.permutation(ids).astype(np.int32))
    indptr = torch.from_numpy(np.sort(np.concatenate([[0], rng.integers(0, n + 1, rows - 1), [n]])).astype(np.int32))
    data = torch.from_numpy(rng.random(n).astype(np.float32) + 0.5)
    grad = torch.from_numpy(rng.standard_normal((rows, dim)).astype(np.float32)).to(dtype)
    row = torch.repeat_interleave(torch.arange(rows), indptr.long().diff())
    at = torch.where(ids < vocab, ids, vocab).long()
    terms = data.double()[:, None] * grad.double()[row]
    want = torch.zeros(vocab + 1, dim, dtype=torch.float64).index_add_(0, at, terms)[:vocab]
    mag = torch.zeros(vocab + 1, dim, dtype=torch.float64).index_add_(0, at, terms.abs())[:vocab]
    most = int(torch.bincount(at).max())
    # `most` fused additions and the joins' at most as many more, each rounding a sum no larger than mag
    e = 2 * most * U * mag
    args = (ids.cuda(), vocab, indptr.cuda(), data.cuda())
    got = dense.embed_rows_grad(grad.cuda(), *args)
    check(got, want, e + half_step(dtype) * (want.abs() + e) + tiny(dtype))
    assert torch.equal(got, dense.embed_rows_grad(grad.cuda(), *args))
    wide = dense.embed_rows_grad(grad.cuda(), *args, dtype=torch.float32)
    check(wide, want, e + half_step(torch.float32) * (want.abs() + e))
    assert torch.equal(wide.to(dtype), got)


@gpu
@pytest.mark.parametrize("dim", [3, 16, 129, 600])
@pytest.mark.parametrize("chunk,longest", [(8, 2300), (16, 9000)])
def test_embed_grad_runs_over_chunks(dim, chunk, longest):
    """Ids that occur so often that their entries, sorted, end just before, at and just behind the ends of 1 .. 10 chunks and of hundreds."""
    rng = np.random.default_rng(dim)
    runs = [c * chunk + d for c in (0, 1, 2, 6, 7, 8, 9, 10) for d in (-1, 0, 1) if c * chunk + d > 0] + [longest] + [1, 2, 3] * 20
    runs += [chunk * 9] * 3 + [chunk] * 5
    ids = np.repeat(np.arange(len(runs)) * 3, runs)
    n, vocab = len(ids), 3 * len(runs)
    assert (2048 < n <= 6144) == (chunk == 8)
    at = rng.permutation(n)
    grad = torch.from_numpy(rng.standard_normal((n, dim)).astype(np.float32))
    idx = torch.from_numpy(ids[at].astype(np.int64))
    want = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, idx, grad.double())
    mag = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, idx, grad.double().abs())
    bound = (2 * torch.bincount(idx, minlength=vocab).double()[:, None] + 1) * U * mag      # an addition an entry, the joins' as many at most, one rounding
    for _ in range(2):
        check(dense.embed_rows_grad(grad.cuda(), idx.cuda(), vocab), want, bound)
    base = torch.ones(vocab, dim, device="cuda")
    dense.embed_rows_grad(grad.cuda(), idx.cuda(), vocab, out=base, accumulate=True)
    check(base, want + 1, bound + U * (mag + 1))
    assert (base[1::3] == 1).all()


@gpu
def test_embed_autograd():
    """The graph's gradient is embed_rows_grad's, also through a broadcast sum, for a table used twice, and against differences."""
    rng = np.random.default_rng(3)
    table = torch.from_numpy(rng.standard_normal((23, 6)).astype(np.float32)).cuda().requires_grad_()
    indptr, ids = csr(rng, 17, 23, 5)
    data = torch.from_numpy(rng.random(ids.numel()).astype(np.float32)).cuda()
    look = torch.from_numpy(rng.integers(0, 23, (3, 4))).cuda()
    weight = torch.from_numpy(rng.standard_normal((17, 6)).astype(np.float32)).cuda()

    def value(t):
        return (dense.embed_rows(t, ids.cuda(), indptr.cuda(), data) * weight).sum() + dense.embed_rows(t, look, scale=2.0).sum()
    value(table).backward()
    want = embed_grad_ref(weight, ids, 23, indptr, data, 1.0)[0] + embed_grad_ref(torch.ones(12, 6), look, 23, None, None, 2.0)[0]
    check(table.grad, want, 1e-5)
    at, step = (4, 2), 0.25                                                       # (linear: a wide step costs nothing)
    with torch.no_grad():
        hi, lo = table.clone(), table.clone()
        hi[at] += step
        lo[at] -= step
        slope = (value(hi) - value(lo)).item() / (2 * step)
    assert abs(slope - table.grad[at].item()) < 1e-3


# ---- score adjustment ------------------------------------------------------------------------------------------------------------

def adjust_ref(scores, targets, history, rep, pres, freq, bias, allowed, filt, target):
    """(result, sum of magnitudes) in 64 bits."""
    n, v = scores.shape
    y, mag = scores.double().cpu().clone(), torch.zeros(n, v, dtype=torch.float64)
    rows = torch.arange(n) if targets is None else targets.long().cpu()

    def counts(c, i):
        out = torch.zeros(v, dtype=torch.int64)
        r = int(rows[i])
        if 0 <= r < c[0].numel() - 1:
            ids = c[1].long().cpu()[int(c[0][r]):int(c[0][r + 1])]
            ids = ids[(ids >= 0) & (ids < v)]
            out += torch.bincount(ids, minlength=v)
        return out

    def of(x, i):
        return float(x.double().reshape(-1)[i]) if torch.is_tensor(x) and x.dim() else float(x)
    for i in range(n):
        # parameters arrive as float32
        r, p, f = (float(np.float32(of(x, i))) for x in (rep, pres, freq))
        c = counts(history, i) if history is not None else torch.zeros(v, dtype=torch.int64)
        hit = c > 0
        y[i] = torch.where(hit, torch.where(y[i] > 0, y[i] / r, y[i] * r), y[i])
        mag[i] = y[i].abs()
        y[i] = torch.where(hit, y[i] - (p + f * c), y[i])
        mag[i] += torch.where(hit, abs(p) + abs(f) * c, 0.0)
        if bias is not None:
            b = (bias if bias.dim() == 1 else bias[i]).double().cpu()
            y[i] += b
            mag[i] += b.abs()
        gone = torch.zeros(v, dtype=torch.bool)
        if filt is not None:
            gone |= counts(filt, i) > 0
        if target is not None:
            gone |= counts(target, i) == 0
        if allowed is not None:
            w = (allowed if allowed.dim() == 1 else allowed[i]).long().cpu()
            gone |= ((w[torch.arange(v) // 32] >> (torch.arange(v) % 32)) & 1) == 0
        y[i][gone] = -math.inf
        mag[i][gone] = 0
    return y, mag


def adjust_bound(y, mag, dtype):
    # quotient or product, the penalty's product and sum, its subtraction, the bias: five roundings of values no larger than mag
    e = 5 * U * mag.nan_to_num(0.0, 0.0, 0.0)
    return e + half_step(dtype) * (torch.where(torch.isfinite(y), y, 0.0).abs() + e) + tiny(dtype)


ADJUST = [  # n, cols, users, mean of history, filter, target; 0: not given
    (1, 1, 1, 1, 0, 0), (3, 31, 4, 6, 3, 9), (2, 32, 2, 40, 0, 0), (5, 33, 9, 0, 5, 0), (4, 1025, 6, 0, 0, 300), (7, 2047, 11, 100, 50, 900),
    (2, 8193, 5, 5000, 3000, 0), (33, 4099, 60, 60, 0, 2000), (300, 9000, 310, 30, 10, 0),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,cols,users,hist,filt,targ", ADJUST)
def test_adjust(dtype, n, cols, users, hist, filt, targ):
    rng = np.random.default_rng(n * 31 + cols)
    it = torch.int64 if n % 2 else torch.int32
    scores = torch.from_numpy(rng.standard_normal((n, cols)) * 3).to(dtype).cuda()
    targets = torch.from_numpy(rng.integers(-1, users + 1, n)).to(it).cuda()
    mk = lambda mean: None if not mean else tuple(t.cuda() for t in csr(rng, users, cols, mean, it, bad=0.1))  # noqa: E731
    h, f, t = mk(hist), mk(filt), mk(targ)
    rep = torch.from_numpy(1 + rng.random(n).astype(np.float32)).cuda()
    pres, freq = torch.from_numpy(rng.random(n).astype(np.float32)).cuda(), 0.125
    bias = torch.from_numpy(rng.standard_normal(cols)).to(TYPES[n % 3]).cuda() if n != 2 else torch.from_numpy(rng.standard_normal((n, cols)).astype(np.float32)).cuda()
    words = torch.from_numpy(rng.integers(-2**31, 2**31, (n, (cols + 31) // 32)).astype(np.int32)).cuda()
    for allowed, tg in ((None, targets), (words, targets), (words[0], None)):
        args = dict(targets=tg, history=h, repetition=rep, presence=pres, frequency=freq, bias=bias, allowed=allowed, filter_cols=f, target_cols=t)
        got = dense.adjust_scores(scores, **args)
        want, mag = adjust_ref(scores, tg, h, rep, pres, freq, bias, allowed, f, t)
        check(got, want, adjust_bound(want, mag, dtype))
        assert torch.equal(got, dense.adjust_scores(scores, **args))
        mine = scores.clone()                                                     # in place
        assert dense.adjust_scores(mine, out=mine, **args).data_ptr() == mine.data_ptr() and torch.equal(mine, got)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_adjust_infinities_nan_and_layouts(dtype):
    """Masked columns become -inf whatever they held; others keep their infinities and NaN; padded rows and what lies beside them."""
    rng = np.random.default_rng(0)
    store = torch.from_numpy(rng.standard_normal((6, 300))).to(dtype).cuda()
    store[:, 40], store[:, 41], store[:, 42] = math.inf, -math.inf, math.nan
    store[:, 50], store[:, 51], store[:, 52] = math.inf, -math.inf, math.nan
    store[:, 60] = torch.finfo(dtype).min
    scores = store[:, 7:280]
    allowed = torch.full((9,), -1, dtype=torch.int32, device="cuda")
    for c in (33, 34, 35, 53):
        allowed[c // 32] &= ~torch.tensor(1 << (c % 32) if c % 32 < 31 else -2**31, dtype=torch.int32, device="cuda")
    h = (torch.tensor([0, 3, 3, 3, 3, 3, 3], device="cuda"), torch.tensor([43, 44, 45], device="cuda"))
    dst = torch.full((6, 290), 3.0, dtype=dtype, device="cuda")
    dense.adjust_scores(scores, history=h, repetition=2.0, allowed=allowed, out=dst[:, 9:282])
    want, mag = adjust_ref(scores, None, h, 2.0, 0.0, 0.0, None, allowed, None, None)
    check(dst[:, 9:282], want, adjust_bound(want, mag, dtype))
    assert (dst[:, :9] == 3).all() and (dst[:, 282:] == 3).all()
    assert (dst[:, 9 + 33:9 + 36] == -math.inf).all() and torch.isnan(dst[:, 9 + 45]).all()
    empty = (torch.zeros(7, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert (dense.adjust_scores(scores, target_cols=empty) == -math.inf).all()    # a mask that leaves nothing
    assert torch.equal(dense.adjust_scores(scores, filter_cols=empty).isnan(), scores.isnan())
    assert dense.adjust_scores(scores[:0]).shape == (0, 273) and dense.adjust_scores(scores[:, :0]).shape == (6, 0)
    wide = store[:1, :273].expand(6, 273)                                         # one row, seen as six
    assert torch.equal(dense.adjust_scores(wide, bias=torch.zeros(273, device="cuda"))[5].nan_to_num(), store[0, :273].nan_to_num())


@gpu
@pytest.mark.parametrize("cols,distinct,entries", [(16_384, 1024, 1600), (16_384, 1025, 3000), (16_384, 1300, 60_000), (16_384, 5000, 65_535), (16_384, 5000, 65_536),
                                                   (16_384, 9000, 70_000), (40_001, 20_000, 40_000), (2048, 2048, 2048), (5000, 1, 2_000_000)])
def test_adjust_long_histories(cols, distinct, entries):
    """Histories at, below and above what a segment's table holds and what 16 bits count: every count is exact, in place as well."""
    rng = np.random.default_rng(entries)
    listed = rng.permutation(cols)[:distinct]
    ids = np.concatenate([listed, rng.choice(listed, entries - distinct)])
    count = torch.from_numpy(np.bincount(ids, minlength=cols))
    indptr = torch.tensor([0, 0, entries], dtype=torch.int32, device="cuda")
    history = (indptr, torch.from_numpy(rng.permutation(ids).astype(np.int32)).cuda())
    scores = torch.zeros(2, cols, device="cuda")
    want = torch.stack([torch.zeros(cols, dtype=torch.int64), -count])              # 0 - 0 - 1 * count, below 2^24: exact
    assert torch.equal(dense.adjust_scores(scores, history=history, frequency=1.0).long().cpu(), want)
    assert torch.equal(dense.adjust_scores(scores, history=history, frequency=1.0, out=scores).long().cpu(), want)


@gpu
def test_adjust_counts_repeats_exactly():
    """A column listed 100 000 times: the count is a whole number, the penalty its exact multiple."""
    scores = torch.zeros(1, 100, device="cuda")
    h = (torch.tensor([0, 100_000], dtype=torch.int32, device="cuda"), torch.full((100_000,), 7, dtype=torch.int32, device="cuda"))
    got = dense.adjust_scores(scores, history=h, frequency=0.5)
    assert got[0, 7].item() == -50_000.0 and got.sum().item() == -50_000.0


# ---- distillation ------------------------------------------------------------------------------------------------------------------

def distill_ref(z, cols, values, counts, tau, tlse, g):
    """(loss, lse, gradient, list mass per row, probabilities on columns, q) in 64 bits, on the CPU."""
    z = z.double().cpu()
    n, v = z.shape
    k = cols.numel() // n
    cols, t = cols.reshape(n, k).long().cpu(), values.reshape(n, k).double().cpu()
    ok = torch.ones(n, k, dtype=torch.bool) if counts is None else torch.arange(k)[None, :] < counts.long().cpu()[:, None]
    ok &= (cols >= 0) & (cols < v)
    t = (t / tau).masked_fill(~ok, -math.inf)
    if tlse is None:
        top = t.max(1, keepdim=True).values if k else torch.full((n, 1), -math.inf, dtype=torch.float64)
        some = top > -math.inf
        logp = torch.where(some, t - top.masked_fill(~some, 0.0), -math.inf)
        logp = logp - torch.log(logp.exp().sum(1, keepdim=True)).masked_fill(~some, 0.0)
    else:
        logp = t - tlse.double().cpu()[:, None]
    p = torch.where(ok, logp.exp(), 0.0)
    lse = torch.logsumexp(z / tau, 1)
    q = torch.where(torch.isneginf(lse)[:, None], 0.0, torch.exp(z / tau - lse[:, None]))
    logq = (z / tau - lse[:, None]).gather(1, cols.clamp(0, v - 1)) if k else torch.zeros(n, 0, dtype=torch.float64)
    loss = tau * tau * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    on = torch.zeros(n, v, dtype=torch.float64)
    if k:
        on.scatter_add_(1, cols.clamp(0, v - 1), p)
    mass = p.sum(1, keepdim=True)
    gg = (torch.ones(n) if g is None else g).double().cpu()[:, None]
    grad = torch.where(mass > 0, gg * tau * (q * mass - on), 0.0)
    return loss, lse, grad, p, on, q, logp, logq


def distill_bounds(z, cols, tau, ref, g, dtype):
    """Bounds of loss and gradient.  c = fl(log2(e) / tau) and z c lie half a step off each: with X the largest |z| log2(e) / tau the exponent of
    2 is off by 3 X u, so every exponential by (3 X + 2) u relatively (v_exp_f32 is good to one step = 2 u).  A thread's sum of its
    share of the columns and the joins add at most (V / 512 + 40) u.  The list: (k + 8 + |log p|) u."""
    loss, lse, grad, p, on, q, logp, logq = ref
    n, v = q.shape
    k = p.shape[1]
    fin = torch.where(torch.isfinite(z.double().cpu()), z.double().cpu(), 0.0).abs()
    x = fin.max(1).values * 1.4427 / tau if v else torch.zeros(n)
    e_q = ((6 * x + 8) + v / 512 + 40)[:, None] * U
    mag = torch.where(p > 0, p * (logp.abs() + logq.abs().nan_to_num(0, 0, 0) + lse.abs().nan_to_num(0, 0, 0)[:, None] + 1), 0.0)
    e_p = (k + 10 + torch.where(p > 0, logp.abs(), 0.0).max(1, keepdim=True).values * 4 if k else torch.zeros(n, 1)) * U
    mass = p.sum(1, keepdim=True)
    loss_b = tau * tau * (mag.sum(1) * (e_p[:, 0] + (k + 8) * U) + mass[:, 0] * e_q[:, 0]) + 1e-30
    gg = (torch.ones(n) if g is None else g).double().cpu().abs()[:, None]
    e = gg * tau * (q * mass * (e_q + e_p + 8 * U) + on * (e_p + 4 * U)) + gg * tau * mass * 2.0 ** -125       # (exponentials below 2^-126 are 0)
    return loss_b, e + half_step(dtype) * (grad.abs() + e) + tiny(dtype)


def lists(rng, n, v, k, distinct=True):
    if distinct:
        cols = np.stack([rng.permutation(v)[:k] for _ in range(n)]) if n else np.zeros((0, k))
    else:
        cols = rng.integers(-2, v + 2, (n, k))
    return torch.from_numpy(cols.astype(np.int64)), torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) * 2 + 3)


DISTILL = [  # rows, columns, slots, temperature, distinct columns
    (1, 1, 1, 1.0, True), (3, 7, 7, 0.5, True), (2, 100, 1, 1.0, True), (5, 333, 20, 2.0, True), (4, 2049, 64, 1.0, False), (9, 4096, 65, 4.0, False),
    (3, 30_011, 200, 1.0, True), (300, 1003, 30, 2.0, False), (257, 9001, 130, 1.0, True), (2, 5000, 4096, 1.0, False),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k,tau,distinct", DISTILL)
@pytest.mark.parametrize("whole", [False, True])
def test_distill(dtype, n, v, k, tau, distinct, whole):
    rng = np.random.default_rng(v + k)
    z = torch.from_numpy(rng.standard_normal((n, v)) * 4).to(dtype).cuda()
    cols, values = lists(rng, n, v, k, distinct)
    counts = torch.from_numpy(rng.integers(0, k + 1, n).astype(np.int32)) if n > 1 else None
    tlse = (torch.logsumexp(values / tau, 1) + 0.3).float() if whole else None
    g = torch.from_numpy(rng.random(n).astype(np.float32) + 0.5)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    cols = cols.to(torch.int32) if n % 2 else cols
    kw = dict(temperature=tau, teacher_lse=dev(tlse))
    args = (dev(cols), dev(values), dev(counts))
    ref = distill_ref(z, cols, values, counts, tau, tlse, g)
    loss_b, grad_b = distill_bounds(z, cols, tau, ref, g, dtype)
    loss, stats = dense.distill_loss(z, *args, return_stats=True, **kw)
    assert loss.dtype == torch.float32 and stats.dtype == torch.float32 and torch.equal(stats[:, 0], z.float().max(1).values)
    check(loss, ref[0], loss_b, "loss")
    check(stats[:, 0].double() / tau + stats[:, 1].double().log(), ref[1], ((6 * (z.double().abs().max().item() * 1.4427 / tau) + 8) + v / 512 + 40) * U, "lse")
    grad = dense.distill_grad(z, stats, *args, grad_loss=dev(g), **kw)
    check(grad, ref[2], grad_b, "grad")
    loss2, grad2 = dense.distill_loss_grad(z, *args, grad_loss=dev(g), **kw)
    check(loss2, ref[0], loss_b, "loss of the one call")
    check(grad2, ref[2], grad_b, "grad of the one call")
    assert torch.equal(grad2, dense.distill_loss_grad(z, *args, grad_loss=dev(g), **kw)[1])
    # in place, and flat lists
    mine = z.clone()
    assert torch.equal(dense.distill_grad(mine, stats, args[0].reshape(-1), args[1].reshape(-1), args[2], grad_loss=dev(g), out=mine, **kw), grad)
    mine = z.clone()
    dense.distill_loss_grad(mine, *args, grad_loss=dev(g), out=mine, **kw)
    assert torch.equal(mine, grad2)


@gpu
@pytest.mark.parametrize("n", [6, 300])
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_masked_scores_and_layouts(dtype, n):
    """Rows of -inf, masked columns, the type's lowest value, a padded row full of NaN with an empty list, teachers of -inf; rows inside a larger store."""
    rng = np.random.default_rng(2)
    v, k = 700, 12
    store = torch.from_numpy(rng.standard_normal((n, v + 31)) * 3).to(dtype)
    z = store[:, 9:9 + v]
    cols, values = lists(rng, n, v, k)
    counts = torch.full((n,), k, dtype=torch.int32)
    z[0, 5:600] = -math.inf                                                       # masked, some of them listed: loss inf
    z[1, :] = -math.inf
    z[2, 100:] = torch.finfo(dtype).min
    z[3, :] = math.nan
    counts[3] = 0
    values[4, 3:] = -math.inf
    values[5, :] = -math.inf
    z[4, 0:300] = -math.inf
    cols[4, :3] = torch.tensor([500, 501, 502])                                    # the list avoids the mask: loss stays finite
    cols[4, 3:] = torch.arange(k - 3)
    store = store.cuda()
    z = store[:, 9:9 + v]
    ref = distill_ref(z, cols, values, counts, 1.0, None, None)
    loss_b, grad_b = distill_bounds(torch.where(z.cpu() < -1e4, torch.zeros((), dtype=dtype), z.cpu()), cols, 1.0, ref, None, dtype)
    args = (cols.cuda(), values.cuda(), counts.cuda())
    want_loss = ref[0].clone()
    want_loss[1] = math.inf                                                       # (log q of a row of -inf only: p log(p / 0))
    want_loss[3] = 0.0
    loss_b[3], grad_b[3] = 0.0, 0.0                                                # an empty list: exactly zero, though the scores are NaN
    # the type's lowest value is finite: its log q is lowest - lse, of which half a step is the bound
    lowest = abs(torch.finfo(dtype).min)
    loss_b[2] = 16 * U * lowest
    want_grad = ref[2].clone()
    want_grad[1] = -ref[4][1]                                                     # q = 0 there
    loss, stats = dense.distill_loss(z, *args, return_stats=True)
    check(loss, want_loss, loss_b, "loss")
    out = torch.full((n, v + 13), 2.0, dtype=dtype, device="cuda")
    dense.distill_grad(z, stats, *args, out=out[:, 5:5 + v])
    check(out[:, 5:5 + v], want_grad, grad_b, "grad")
    assert (out[:, :5] == 2).all() and (out[:, 5 + v:] == 2).all()
    check(dense.distill_loss_grad(z, *args)[1], want_grad, grad_b, "grad of the one call")
    assert (out[3, 5:5 + v] == 0).all() and (out[5, 5:5 + v] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,tau", [(2, 700, 1.0), (300, 700, 1.0), (2, 9000, 0.25)])
def test_distill_row_of_the_lowest_value(dtype, n, v, tau):
    """Every score masked with the type's lowest (or highest) finite value: q is uniform over the columns that hold it."""
    z = torch.full((n, v), torch.finfo(dtype).min, dtype=dtype)
    z[1] = torch.randn(v, generator=torch.Generator().manual_seed(0)).to(dtype)
    z[1, 7] = torch.finfo(dtype).max
    cols, values = torch.tensor([[3, 7]]).repeat(n, 1), torch.tensor([[1.0, 1.0]]).repeat(n, 1)
    loss, grad = dense.distill_loss_grad(z.cuda(), cols.cuda(), values.cuda(), temperature=tau)
    loss2, stats = dense.distill_loss(z.cuda(), cols.cuda(), values.cuda(), temperature=tau, return_stats=True)
    grad2 = dense.distill_grad(z.cuda(), stats, cols.cuda(), values.cuda(), temperature=tau)
    q = torch.full((n, v), 1.0 / v, dtype=torch.float64)
    q[1] = 0.0
    q[1, 7] = 1.0
    want = tau * q
    want[:, 3] -= tau / 2
    want[:, 7] -= tau / 2
    flat = torch.full((n,), tau * tau * (math.log(0.5) + math.log(v)), dtype=torch.float64)
    for a in (loss, loss2):
        check(a[[0] + list(range(2, n))], flat[1:], 40 * U * 10)
    for a in (grad, grad2):
        check(a, want, 40 * U + half_step(dtype) * (want.abs() + 40 * U) + tiny(dtype))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(300, 4099), (300, 4103), (5, 4103), (260, 7), (260, 40_013)])
def test_distill_every_listed_place(dtype, n, v):
    """Listed columns at the row's first and last places, at the borders of vectors and pieces, named once, twice and many times: each is
    written after the vector it lies in."""
    rng = np.random.default_rng(v)
    k = 64
    places = np.concatenate([np.arange(v - min(v, 12), v), np.arange(min(v, 9)), [v // 2, v // 2, v // 2 + 1], rng.integers(0, v, k)])[:k]
    cols = torch.from_numpy(np.stack([rng.permutation(places) for _ in range(n)]).astype(np.int64))
    cols[1] = v - 1                                                               # one column, k times
    values = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32))
    z = torch.from_numpy(rng.standard_normal((n, v)) * 2).to(dtype).cuda()
    ref = distill_ref(z, cols, values, None, 1.0, None, None)
    grad_b = distill_bounds(z, cols, 1.0, ref, None, dtype)[1]
    loss, stats = dense.distill_loss(z, cols.cuda(), values.cuda(), return_stats=True)
    check(dense.distill_grad(z, stats, cols.cuda(), values.cuda()), ref[2], grad_b)
    for _ in range(3):
        check(dense.distill_loss_grad(z, cols.cuda(), values.cuda())[1], ref[2], grad_b)


@gpu
@pytest.mark.parametrize("n", [257, 5])
@pytest.mark.parametrize("dtype,v,k", [(torch.float32, 150_001, 3), (torch.float32, 110_003, 4096), (torch.bfloat16, 300_007, 300), (torch.float16, 131_072, 64)])
def test_distill_rows_longer_than_a_workgroup_keeps(dtype, v, k, n):
    """The one call on rows that do not fit registers and LDS (their rest is read twice, or few of them are cut into pieces), in place as well,
    next to the two calls."""
    some = [0, n // 2, n - 1]
    gen = torch.Generator(device="cuda").manual_seed(v)
    z = (torch.randn(n, v, generator=gen, device="cuda") * 2).to(dtype)
    cols = torch.randint(0, v, (n, k), generator=gen, device="cuda")
    cols[:, :2] = torch.tensor([v - 1, v - 40], device="cuda")
    values = torch.randn(n, k, generator=gen, device="cuda")
    ref = distill_ref(z[some], cols[some].cpu(), values[some].cpu(), None, 1.0, None, None)
    loss_b, grad_b = distill_bounds(z[some], cols[some].cpu(), 1.0, ref, None, dtype)
    loss, stats = dense.distill_loss(z, cols, values, return_stats=True)
    check(loss[some], ref[0], loss_b, "loss")
    check(dense.distill_grad(z, stats, cols, values)[some], ref[2], grad_b, "grad")
    loss, grad = dense.distill_loss_grad(z, cols, values)
    check(loss[some], ref[0], loss_b, "loss of the one call")
    check(grad[some], ref[2], grad_b, "grad of the one call")
    assert torch.equal(dense.distill_loss_grad(z, cols, values, out=z)[1], grad) and torch.equal(z, grad)


@gpu
@pytest.mark.parametrize("dtype,v", [(torch.float32, 120_001), (torch.bfloat16, 400_003), (torch.float16, 220_000)])
def test_distill_masked_pieces(dtype, v):
    """Rows long enough to be cut: pieces that are -inf altogether, one column left, the lowest value everywhere, a padded row of NaN, a row of -inf."""
    rng = np.random.default_rng(v)
    n, k = 5, 9
    z = torch.from_numpy(rng.standard_normal((n, v)).astype(np.float32) * 3).to(dtype)
    cols, values = lists(rng, n, v, k)
    counts = torch.full((n,), k, dtype=torch.int32)
    z[0, : v * 2 // 3] = -math.inf
    cols[0] = torch.arange(v - k, v)
    z[1, :] = -math.inf
    z[1, v - 3] = 1.5
    counts[1], cols[1, 0] = 1, v - 3                                               # p = q = 1 there
    z[2, :] = torch.finfo(dtype).min
    z[3, :] = math.nan
    counts[3] = 0
    z[4, :] = -math.inf
    ref = distill_ref(z, cols, values, counts, 1.0, None, None)
    loss_b, grad_b = distill_bounds(torch.where(z < -1e4, torch.zeros((), dtype=dtype), z), cols, 1.0, ref, None, dtype)
    want_loss, want_grad = ref[0].clone(), ref[2].clone()
    want_loss[3], want_loss[4], loss_b[3], grad_b[3] = 0.0, math.inf, 0.0, 0.0
    want_grad[3], want_grad[4] = 0.0, -ref[4][4]                                   # a row of -inf only has q = 0
    # the lowest value everywhere: q = 1 / v, which lowest + log v does not tell in 64 bits either (2^128 against log v < 2^4)
    logp, p = ref[6][2], ref[3][2]
    want_loss[2] = torch.where(p > 0, p * (logp + math.log(v)), 0.0).sum()
    want_grad[2] = 1.0 / v - ref[4][2]
    loss_b[2], grad_b[2] = 400 * U, 40 * U + half_step(dtype) * (want_grad[2].abs() + 40 * U) + tiny(dtype)
    z, args = z.cuda(), (cols.cuda(), values.cuda(), counts.cuda())
    loss, stats = dense.distill_loss(z, *args, return_stats=True)
    check(loss, want_loss, loss_b, "loss")
    check(dense.distill_grad(z, stats, *args), want_grad, grad_b, "grad")
    loss, grad = dense.distill_loss_grad(z, *args)
    check(loss, want_loss, loss_b, "loss of the one call")
    check(grad, want_grad, grad_b, "grad of the one call")
    assert torch.equal(dense.distill_loss_grad(z, *args, out=z)[1], grad)


@gpu
def test_distill_sizes_of_nothing():
    z = torch.randn(3, 50, device="cuda")
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    loss, grad = dense.distill_loss_grad(z, none, torch.zeros(3, 0, device="cuda"))
    assert (loss == 0).all() and (grad == 0).all() and grad.shape == z.shape
    assert dense.distill_loss(z[:0], none[:0], torch.zeros(0, 0, device="cuda")).shape == (0,)
    one = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    loss, stats = dense.distill_loss(z[:, :0], one, torch.ones(3, 1, device="cuda"), return_stats=True)      # no columns: no id is inside
    assert (loss == 0).all() and (stats[:, 0] == -math.inf).all() and (stats[:, 1] == 0).all()


@gpu
def test_distill_autograd():
    """The graph's gradient against the formula and against differences."""
    rng = np.random.default_rng(8)
    n, v, k = 4, 60, 5
    z = torch.from_numpy(rng.standard_normal((n, v)).astype(np.float32)).cuda().requires_grad_()
    cols, values = (t.cuda() for t in lists(rng, n, v, k))
    w = torch.tensor([0.5, 1.0, 2.0, 0.0], device="cuda")
    (dense.distill_loss(z, cols, values, temperature=2.0) * w).sum().backward()
    ref = distill_ref(z.detach(), cols, values, None, 2.0, None, w)
    check(z.grad, ref[2], distill_bounds(z.detach(), cols, 2.0, ref, w, torch.float32)[1])
    z2 = z.detach().clone().requires_grad_()
    dense.distill_loss(z2, cols, values, temperature=2.0).mean().backward()       # a broadcast gradient
    check(z2.grad, distill_ref(z.detach(), cols, values, None, 2.0, None, torch.full((n,), 0.25))[2], 1e-6)
    step = 1e-2
    for at in ((0, int(cols[0, 0])), (1, 7)):
        hi, lo = z.detach().clone(), z.detach().clone()
        hi[at] += step
        lo[at] -= step
        slope = ((dense.distill_loss(hi, cols, values, temperature=2.0) - dense.distill_loss(lo, cols, values, temperature=2.0)) * w).sum().item() / (2 * step)
        # third derivatives are below tau^2 / tau^3: step^2 / 6 of that, and the losses' own rounding over the step
        assert abs(slope - z.grad[at].item()) < 5e-4


# ---- as they are used: streams, graphs, together ------------------------------------------------------------------------------------

@gpu
def test_run_together():
    """Histories -> user vectors -> scores -> divergence from the neighbourhood model's own lists -> gradient of the table; then
    the served scores, seen items dropped with the selectors of the similarity functions."""
    import scipy.sparse as sp

    from similaripy_amd import _host
    from similaripy_amd.device import DeviceProblem
    rng = np.random.default_rng(21)
    urm = sp.random_array((300, 500), density=0.03, format="csr", dtype=np.float32, random_state=rng)
    sim = sp.random_array((500, 500), density=0.05, format="csr", dtype=np.float32, random_state=rng)
    call = _host.prepare(urm, sim, k=20, filter_cols=urm)
    prob = DeviceProblem(call)
    cols, vals, counts, _ = prob.alloc_outputs()
    prob.run(cols, vals, counts)
    table = (torch.randn(500, 48, device="cuda") * 0.1).requires_grad_()
    users = prob.embed(table)
    scores = users @ table.detach().T
    loss = prob.distill_loss(scores, cols, vals, counts, temperature=0.5)
    loss.mean().backward()
    # the same in 64 bits on the CPU
    t = table.detach().double().cpu().requires_grad_()
    m1 = torch.from_numpy(urm.toarray()).double()
    z = (m1 @ t) @ t.detach().T
    ok = torch.arange(20)[None, :] < counts.cpu()[:, None]
    v = (vals.view(300, 20).double().cpu() / 0.5).masked_fill(~ok, -math.inf)
    logp = torch.where(ok.any(1, keepdim=True), v, torch.zeros_like(v)).log_softmax(1)
    p = torch.where(ok, logp.exp(), 0.0)
    logq = (z / 0.5).log_softmax(1).gather(1, cols.view(300, 20).long().cpu())
    ref = 0.25 * torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
    ref.mean().backward()
    check(loss, ref, 1e-5 * (ref.detach().abs() + 1))
    check(table.grad, t.grad, 1e-4 * t.grad.abs().max())
    seen = prob.adjust_scores(scores.detach())
    assert torch.equal(torch.isneginf(seen).cpu(), torch.from_numpy(urm.toarray() != 0))
    some = torch.tensor([7, 299, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(prob.adjust_scores(scores.detach()[some.long()], targets=some), seen[some.long()])


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in the table, its gradient, the scores: the last rows are where they belong."""
    vocab, dim = 2_200_000, 1024
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(dim, device="cuda").to(torch.bfloat16)
    table[-1], table[0] = last, 3.0
    ids = torch.tensor([vocab - 1, 0, vocab - 1], device="cuda")
    assert torch.equal(dense.embed_rows(table, ids)[2], last)
    bag = dense.embed_rows(table, ids, torch.tensor([0, 1, 3], device="cuda"))
    assert torch.equal(bag[0], last) and torch.equal(bag[1], (last.float() + 3.0).to(torch.bfloat16))
    for n in (3, 3000, 12_000):                                                   # without a sort, by one workgroup, by all
        many = ids.repeat(n // 3)
        grad = dense.embed_rows_grad(torch.ones(n, dim, dtype=torch.bfloat16, device="cuda"), many, vocab, out=table)
        assert (grad[-1] == float(n // 3 * 2)).all() and (grad[0] == float(n // 3)).all() and grad[1:-1:100_003].abs().max() == 0
        assert grad[-2].abs().max() == 0
    del table, grad
    n, v = 27_000, 80_000
    z = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    z[-1, -1], z[-1, 5] = 2.0, -1.0
    one = (torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([v - 1, 5], dtype=torch.int32, device="cuda"))
    where = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    where[-1] = 0
    out = dense.adjust_scores(z, targets=where, history=one, repetition=4.0, out=z)
    assert out[-1, -1].item() == 0.5 and out[-1, 5].item() == -4.0 and out[-1].count_nonzero().item() == 2 and out[0].count_nonzero().item() == 0
    cols, values = torch.full((n, 1), v - 1, dtype=torch.int32, device="cuda"), torch.ones(n, 1, device="cuda")
    row = z[-1].double().cpu()
    loss, stats = dense.distill_loss(z, cols, values, return_stats=True)
    assert abs(loss[-1].item() + (row[-1] - torch.logsumexp(row, 0)).item()) < 1e-4
    want = torch.softmax(row, 0)
    want[-1] -= 1.0
    for grad in (dense.distill_grad(z, stats, cols, values, out=z.clone()), dense.distill_loss_grad(z, cols, values, out=z)[1]):
        check(grad[-1], want, 2.0 ** -8 * want.abs() + 1e-8)


@gpu
def test_captured_large_rows():
    """The kernel that keeps a row in LDS beyond what every kernel may have, and the sorted gradient, replayed."""
    n, v = 300, 90_000
    z = torch.randn(n, v, device="cuda")
    cols, values = torch.randint(0, v, (n, 10), device="cuda"), torch.randn(n, 10, device="cuda")
    ids, grad = torch.randint(0, 5000, (20_000,), device="cuda"), torch.randn(20_000, 30, device="cuda")

    def both():
        return (*dense.distill_loss_grad(z, cols, values), dense.embed_rows_grad(grad, ids, 5000))
    both()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = both()
    for seed in range(3):
        for t in (z, grad):
            t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        g.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


@gpu
def test_embed_shapes_of_nothing():
    """Rows without columns, a single id without dimensions, through the graph as well."""
    table = torch.zeros(5, 0, device="cuda", requires_grad=True)
    out = dense.embed_rows(table, torch.zeros(2, 3, dtype=torch.int64, device="cuda"))
    assert out.shape == (2, 3, 0)
    out.sum().backward()
    assert table.grad.shape == (5, 0)
    table = torch.arange(12.0, device="cuda").view(4, 3).requires_grad_()
    out = dense.embed_rows(table, torch.tensor(2, device="cuda"))
    assert out.shape == (3,)
    out.sum().backward()
    assert table.grad[2].tolist() == [1.0, 1.0, 1.0] and table.grad.sum().item() == 3.0


@gpu
def test_replayed_graphs_share_nothing():
    """Two captured graphs, replayed alternately with eager work between them, give the eager results every time."""
    rng = np.random.default_rng(4)
    n, v, d = 12, 5000, 40
    table, z = torch.randn(v, d, device="cuda"), torch.randn(n, v, device="cuda")
    ids = torch.from_numpy(rng.integers(0, v, 3000)).cuda()
    grad = torch.randn(3000, d, device="cuda")
    cols, values = (t.cuda() for t in lists(rng, n, v, 30))
    h = tuple(t.cuda() for t in csr(rng, n, v, 50))

    def one():
        return dense.embed_rows(table, ids), dense.embed_rows_grad(grad, ids, v), dense.adjust_scores(z, history=h, repetition=1.5, filter_cols=h)

    def two():
        loss, stats = dense.distill_loss(z, cols, values, return_stats=True)
        return loss, dense.distill_grad(z, stats, cols, values), dense.distill_loss_grad(z, cols, values)[1]
    one(), two()
    torch.cuda.synchronize()
    graphs = []
    for f in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = f()
        graphs.append((g, res, f))
    for turn in range(4):
        for t in (table, z, grad):
            t.copy_(torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(turn), device="cuda"))
        for g, res, f in graphs if turn % 2 else graphs[::-1]:
            g.replay()
            want = f()
            torch.cuda.synchronize()
            for a, b in zip(res, want):
                assert torch.equal(a, b)


@gpu
def test_autograd_refuses_capture():
    table = torch.randn(10, 4, device="cuda", requires_grad=True)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="cannot be captured"):
            dense.embed_rows(table, ids)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            dense.distill_loss(table, torch.zeros(10, 1, dtype=torch.int32, device="cuda"), torch.zeros(10, 1, device="cuda"))
        dense.embed_rows(table.detach(), ids)


@gpu
def test_other_stream():
    table, ids = torch.randn(1000, 64, device="cuda"), torch.arange(1000, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = [dense.embed_rows(table, ids, scale=float(i)) for i in range(20)]
        grads = [dense.embed_rows_grad(o, ids, 1000) for o in out]
    torch.cuda.current_stream().wait_stream(s)
    for i, (o, g) in enumerate(zip(out, grads)):
        assert torch.equal(o, table * i) and torch.equal(g, o)


@gpu
def test_two_threads_at_once():
    """Calls from two threads, each on a stream of its own."""
    import threading
    rng = np.random.default_rng(6)
    n, v = 40, 3000
    z = torch.from_numpy(rng.standard_normal((n, v)).astype(np.float32)).cuda()
    cols, values = (t.cuda() for t in lists(rng, n, v, 20))
    ids = torch.from_numpy(rng.integers(0, v, 4000)).cuda()
    g = torch.randn(4000, 33, device="cuda")
    want = (dense.distill_loss_grad(z, cols, values)[1], dense.embed_rows_grad(g, ids, v))
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = (dense.distill_loss_grad(z, cols, values)[1], dense.embed_rows_grad(g, ids, v))
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)
    threads = [threading.Thread(target=work) for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


# ---- refusals (CPU) ------------------------------------------------------------------------------------------------------------------

def _struct_fields(name):
    body = HEADER[HEADER.index("typedef struct %s {" % name):]
    body = re.sub(r"/\*.*?\*/", "", body[body.index("{") + 1:body.index("} %s;" % name)], flags=re.S)
    names = []
    for stmt in filter(None, (s.strip() for s in body.split(";"))):
        first, *rest = stmt.split(",")
        names += [first.split()[-1].lstrip("*")] + [r.strip().lstrip("*") for r in rest]
    return names


@pytest.mark.parametrize("name,mirror", [("sp_embed_args", _abi.SpEmbedArgs), ("sp_csr_pattern", _abi.SpCsrPattern), ("sp_adjust_args", _abi.SpAdjustArgs),
                                         ("sp_distill_args", _abi.SpDistillArgs)])
def test_structs_mirror_the_header(name, mirror):
    assert _struct_fields(name) == [f[0] for f in mirror._fields_]


def test_every_declared_symbol_is_exported():
    declared = set(re.findall(r"^\s*(?:int64_t|int)\s+(sp_[a-z0-9_]+)\s*\(", HEADER, flags=re.M))
    assert declared == set(_abi.DENSE_SYMBOLS)
    lib = _abi.load()
    assert all(getattr(lib, s) is not None for s in declared)


def _c(symbol, args, size=True):
    import ctypes as C
    if size:
        args.struct_size = C.sizeof(args)
    return getattr(_abi.load(), symbol)(C.byref(args)), _abi.last_error()


def test_c_entries_refuse():
    """Bad sizes, types and pointers are turned down before any device is asked for."""
    for symbol, cls in (("sp_embed_rows", _abi.SpEmbedArgs), ("sp_embed_rows_grad", _abi.SpEmbedArgs), ("sp_adjust_scores", _abi.SpAdjustArgs),
                        ("sp_distill_loss", _abi.SpDistillArgs), ("sp_distill_grad", _abi.SpDistillArgs), ("sp_distill_loss_grad", _abi.SpDistillArgs)):
        a = cls()
        a.struct_size = 8
        rc, err = _c(symbol, a, size=False)
        assert rc == -1 and "size mismatch" in err
        a = cls()
        a.flags = 1
        assert _c(symbol, a)[0] == -1
        a = cls()
        a.dtype = 3
        assert _c(symbol, a)[0] == -1
        a = cls()
        a.n_rows = -1
        assert _c(symbol, a)[0] == -1
    e = _abi.SpEmbedArgs()
    e.n_rows, e.nnz, e.dim, e.n_vocab = 4000, 3999, 2, 5
    assert "nnz must equal n_rows" in _c("sp_embed_rows", e)[1]
    e.nnz = 4000
    assert "NULL indices" in _c("sp_embed_rows", e)[1]
    e.indices = 64
    assert "NULL table" in _c("sp_embed_rows", e)[1]
    e.src, e.out, e.ld_out = 64, 64, 1
    assert "overlap" in _c("sp_embed_rows", e)[1]
    e.ld_out = 2
    rc, err = _c("sp_embed_rows_grad", e)
    assert rc == -5 and "workspace too small" in err
    assert _c("sp_embed_rows_grad_workspace_bytes", e)[0] > 0
    e.n_vocab = 2**31 - 1
    assert _c("sp_embed_rows_grad", e)[0] == -1
    d = _abi.SpDistillArgs()
    d.n_rows, d.n_cols, d.k, d.temperature = 2**23, 3, 1, 1.0                        # more threads than a launch can have
    assert "too many rows" in _c("sp_distill_loss", d)[1]
    d.n_rows, d.n_cols, d.k = 2, 2**31 - 1, 1
    assert "bad shape" in _c("sp_distill_loss", d)[1]
    d.n_rows, d.n_cols, d.k, d.temperature = 2, 3, 4097, 0.0
    assert "k = 4097" in _c("sp_distill_loss", d)[1]
    d.k = 1
    for t in (0.0, -1.0, math.nan, math.inf):
        d.temperature = t
        assert "temperature" in _c("sp_distill_loss", d)[1]
    d.temperature = 1.0
    assert "NULL" in _c("sp_distill_loss", d)[1]
    d.student = d.cols = d.values = 64
    d.n_cols = 1 << 20                                                             # (rows in pieces: their sums need a workspace)
    assert _c("sp_distill_loss", d)[0] == -5
    assert "grad is NULL" in _c("sp_distill_grad", d)[1]
    d.grad = 64
    assert "stats is NULL" in _c("sp_distill_grad", d)[1]
    s = _abi.SpAdjustArgs()
    s.n_rows, s.n_cols = 2, 3
    assert "NULL scores" in _c("sp_adjust_scores", s)[1]
    s.history.indptr, s.history.nnz = 64, 3
    assert "history" in _c("sp_adjust_scores", s)[1]


@pytest.mark.skipif(_abi.device_count() > 0, reason="only meaningful on a box without a GPU")
def test_no_cpu_fallback():
    e = _abi.SpEmbedArgs()
    e.n_rows = e.nnz = 1
    e.n_vocab = e.dim = e.ld_out = e.ld_src = 1
    e.indices = e.src = e.out = 64
    rc, err = _c("sp_embed_rows", e)
    assert rc == -2 and "no CPU fallback" in err
    for f in (lambda: dense.embed_rows(torch.zeros(2, 2), torch.zeros(1, dtype=torch.int64)), lambda: dense.adjust_scores(torch.zeros(2, 2)),
              lambda: dense.distill_loss(torch.zeros(2, 2), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1)),
              lambda: dense.embed_rows_grad(torch.zeros(1, 2), torch.zeros(1, dtype=torch.int64), 3)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            f()


def test_wrong_operands():
    with pytest.raises(TypeError):
        dense.embed_rows(np.zeros((2, 2)), None)
    with pytest.raises(TypeError):
        dense.adjust_scores(torch.zeros(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError):
        dense.adjust_scores(torch.zeros(2))


@gpu
def test_wrong_operands_on_a_device():
    z = torch.zeros(4, 6, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    i32 = torch.zeros(4, dtype=torch.int32, device="cuda")
    cols, vals = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda")
    leaf = torch.zeros(4, 6, device="cuda", requires_grad=True)
    bad = [
        lambda: dense.embed_rows(z.T, ids), lambda: dense.embed_rows(z, ids.float()), lambda: dense.embed_rows(z, ids.cpu()),
        lambda: dense.embed_rows(z, ids, i32), lambda: dense.embed_rows(z, ids, None, vals), lambda: dense.embed_rows(z, ids, ids, vals[0, :1]),
        lambda: dense.embed_rows(z, ids, ids, torch.zeros(3, device="cuda").double()), lambda: dense.embed_rows(z, ids, out=z[:3]),
        lambda: dense.embed_rows(z, ids, out=z.new_zeros(3, 5)), lambda: dense.embed_rows(z, ids.reshape(3, 1), ids),
        lambda: dense.embed_rows_grad(z, ids, 5), lambda: dense.embed_rows_grad(z[:3], ids, -1), lambda: dense.embed_rows_grad(z[:3], ids, 5, accumulate=True),
        lambda: dense.embed_rows_grad(z[:3], ids, 5, dtype=torch.float16), lambda: dense.embed_rows_grad(z[:3], ids, 4, out=z),
        lambda: dense.embed_rows_grad(z[:3], ids, 5, out=z.new_zeros(1, 6).expand(5, 6)),
        lambda: dense.adjust_scores(z, targets=ids), lambda: dense.adjust_scores(z, history=i32), lambda: dense.adjust_scores(z, history=(i32, ids)),
        lambda: dense.adjust_scores(z, repetition=0.0), lambda: dense.adjust_scores(z, repetition=torch.ones(3, device="cuda")),
        lambda: dense.adjust_scores(z, bias=torch.zeros(5, device="cuda")), lambda: dense.adjust_scores(z, allowed=torch.zeros(2, dtype=torch.int32, device="cuda")),
        lambda: dense.adjust_scores(z, allowed=torch.zeros(1, dtype=torch.int64, device="cuda")), lambda: dense.adjust_scores(z[:3], out=z[1:]),
        lambda: dense.adjust_scores(z.requires_grad_()),
        lambda: dense.distill_loss(z.detach(), cols[:3], vals), lambda: dense.distill_loss(z.detach(), cols, vals[:3]), lambda: dense.distill_loss(z.detach(), cols, vals, ids),
        lambda: dense.distill_loss(z.detach(), cols, vals, i32[:3]), lambda: dense.distill_loss(z.detach(), cols, vals, temperature=0.0),
        lambda: dense.distill_loss(z.detach(), cols, vals, temperature=math.nan), lambda: dense.distill_loss(z.detach(), cols, vals.double()),
        lambda: dense.distill_loss(z.detach(), torch.zeros(4, 4097, dtype=torch.int32, device="cuda"), torch.zeros(4, 4097, device="cuda")),
        lambda: dense.distill_loss(z.detach(), cols, vals.clone().requires_grad_()), lambda: dense.distill_loss(leaf, cols, vals.clone().requires_grad_()),
        lambda: dense.distill_loss(leaf, cols, vals, teacher_lse=torch.zeros(4, device="cuda").requires_grad_()),
        lambda: dense.embed_rows(leaf, ids, torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(3, device="cuda").requires_grad_()),
        lambda: dense.adjust_scores(z, repetition=torch.tensor(0.0)), lambda: dense.distill_loss(z.detach(), cols, vals.T.contiguous()), lambda: dense.embed_rows(z, ids, out=[1]), lambda: dense.distill_grad(z.detach(), torch.zeros(4, device="cuda"), cols, vals),
        lambda: dense.distill_loss_grad(z.detach(), cols, vals, grad_loss=torch.zeros(3, device="cuda")), lambda: dense.distill_loss(z.detach(), cols.T, vals.T),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            f()
            raise AssertionError(f"call {i} went through")
