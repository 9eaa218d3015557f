"""Calls of the dense operators that tests/test_dense.py does not make: what the documentation allows and what it refuses.

u = 2^-24 is half a step of float32, as there.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from similaripy_amd import dense
from tests.test_dense import TYPES, U, check, distill_bounds, distill_ref

gpu = pytest.mark.gpu


# ---- distillation: scores far from 0 -------------------------------------------------------------------------------------------

def masked_row(kind, z, mask, v):
    """A row in which `mask` stands where nothing may be chosen; the columns of its list are among the last three."""
    if kind == "all":
        z[:] = mask
    elif kind == "most":
        z[: v - 40] = mask
    elif kind == "one":
        z[: v - 1] = mask
    else:                                               # in stripes, so that a thread meets the mask before and after scores
        z[::2] = mask
        z[v - 3:] = 1.0


@gpu
@pytest.mark.parametrize("n,v", [(5, 700), (5, 9001), (300, 9001), (5, 120_001), (260, 120_001)])
@pytest.mark.parametrize("dtype,mask,tau", [
    (torch.float32, -1e9, 1.0), (torch.float32, -1e10, 1.0), (torch.float32, -1e20, 1.0), (torch.float32, -1e30, 1.0), (torch.float32, -1e30, 0.07),
    (torch.float32, None, 2.0), (torch.float32, None, 3.0), (torch.float32, -2e9, 1.0), (torch.bfloat16, -1e10, 1.0), (torch.bfloat16, -1e30, 1.0),
    (torch.bfloat16, None, 2.0), (torch.bfloat16, None, 10.0), (torch.float16, None, 2e-5), (torch.float32, 1e12, 1.0)])
def test_distill_masks_of_any_size(dtype, mask, tau, n, v):
    """Finite masks between the scores and the type's lowest value (None), over rows, most of a row, every other column; also scores that are
    all large (a positive "mask": the columns that hold it share the probability)."""
    rng = np.random.default_rng(v)
    mask = torch.finfo(dtype).min if mask is None else mask
    z = torch.from_numpy(rng.standard_normal((n, v)).astype(np.float32)).to(dtype)
    for i, kind in enumerate(("all", "most", "one", "stripes")):
        masked_row(kind, z[i], mask, v)
    cols = torch.tensor([v - 1, v - 3, v - 2]).repeat(n, 1)
    cols[2] = v - 1
    values = torch.from_numpy(rng.standard_normal((n, 3)).astype(np.float32))
    if mask > 0:                                        # the list names columns of the maximum
        z[1, v - 3:], z[2, v - 1], z[3, v - 3:] = mask, mask, mask
    some = [0, 1, 2, 3, 4]
    # the softmax does not change when the row's maximum is taken off, which is exact enough in 64 bits
    shifted = z[some].double() - z[some].double().max(1, keepdim=True).values
    ref = distill_ref(shifted, cols[some], values[some], None, tau, None, None)
    loss_b, grad_b = distill_bounds(torch.where(shifted < -1e4, 0.0, shifted), cols[some], tau, ref, None, dtype)
    # the rounded exponent and its correction are up to 64 each on top of what distill_bounds counts
    mass = ref[3].sum(1)
    loss_b, grad_b = loss_b + tau * tau * mass * 2 * 64 * U, grad_b + tau * ref[5] * mass[:, None] * 2 * 64 * U
    z, args = z.cuda(), (cols.cuda(), values.cuda())
    loss, stats = dense.distill_loss(z, *args, temperature=tau, return_stats=True)
    check(loss[some], ref[0], loss_b, "loss")
    check(dense.distill_grad(z, stats, *args, temperature=tau)[some], ref[2], grad_b, "grad")
    loss, grad = dense.distill_loss_grad(z, *args, temperature=tau)
    check(loss[some], ref[0], loss_b, "loss of the one call")
    check(grad[some], ref[2], grad_b, "grad of the one call")
    assert not loss.isnan().any() and not grad.isnan().any()
    assert torch.equal(dense.distill_loss_grad(z, *args, temperature=tau, out=z)[1], grad)


# ---- what torch has to know: changed outputs, tangents, traces --------------------------------------------------------------------

def small(device):
    """A call of every function, as (function of named operands, its float operands)."""
    z = torch.randn(3, 8, device=device)
    ids = torch.tensor([0, 2, 1], device=device)
    ptr = torch.tensor([0, 1, 3], device=device)
    w = torch.ones(3, device=device)
    cols, values = torch.tensor([[0, 1]] * 3, device=device), torch.randn(3, 2, device=device)
    stats, row = torch.ones(3, 2, device=device), torch.zeros(8, device=device)
    history = (torch.tensor([0, 1, 1, 1], device=device), ids[:1])
    return {
        "embed_rows": (lambda table, data: dense.embed_rows(table, ids, ptr, data), {"table": z, "data": w}),
        "embed_rows out": (lambda out: dense.embed_rows(z, ids, out=out), {"out": torch.empty(3, 8, device=device)}),
        "embed_rows_grad": (lambda grad, data: dense.embed_rows_grad(grad, ids, 5, ptr, data), {"grad": z[:2].clone(), "data": w}),
        "embed_rows_grad out": (lambda out: dense.embed_rows_grad(z, ids, 3, out=out), {"out": torch.empty(3, 8, device=device)}),
        "adjust_scores": (lambda scores, bias, repetition, presence, frequency: dense.adjust_scores(
            scores, history=history, bias=bias, repetition=repetition, presence=presence, frequency=frequency),
            {"scores": z, "bias": torch.zeros(8, device=device), "repetition": w, "presence": w, "frequency": w}),
        "adjust_scores out": (lambda out: dense.adjust_scores(z, bias=row, out=out), {"out": torch.empty(3, 8, device=device)}),
        "distill_loss": (lambda student, values, teacher_lse: dense.distill_loss(student, cols, values, teacher_lse=teacher_lse),
                         {"student": z, "values": values, "teacher_lse": w * 2}),
        "distill_grad": (lambda student, stats, values, grad_loss: dense.distill_grad(student, stats, cols, values, grad_loss=grad_loss),
                         {"student": z, "stats": stats, "values": values, "grad_loss": w}),
        "distill_grad out": (lambda out: dense.distill_grad(z, stats, cols, values, out=out), {"out": torch.empty(3, 8, device=device)}),
        "distill_loss_grad": (lambda student, values, grad_loss, teacher_lse: dense.distill_loss_grad(
            student, cols, values, grad_loss=grad_loss, teacher_lse=teacher_lse), {"student": z, "values": values, "grad_loss": w, "teacher_lse": w}),
        "distill_loss_grad out": (lambda out: dense.distill_loss_grad(z, cols, values, out=out), {"out": torch.empty(3, 8, device=device)}),
    }


CALLS = list(small("cpu"))
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


@gpu
@pytest.mark.parametrize("name", [c for c in CALLS if c.endswith(" out")])
def test_outputs_count_as_changed(name):
    """A tensor that an autograd graph has saved may be written by a call, but not unnoticed: its version goes up, also through views."""
    fn, operands = small("cuda")[name]
    out = operands["out"]
    before, row = out._version, out[1]
    fn(**operands)
    assert out._version > before and row._version == out._version
    with torch.inference_mode():                        # (tensors made there have no version)
        fn, operands = small("cuda")[name]
        fn(**operands)


@gpu
def test_backward_of_an_overwritten_student():
    """The backward pass needs the scores: overwritten in place meanwhile, it raises as it does for torch's own operators."""
    leaf = torch.randn(3, 50, device="cuda", requires_grad=True)
    cols, values = torch.tensor([[0, 1]] * 3, device="cuda"), torch.randn(3, 2, device="cuda")
    scores = leaf * 1.0
    loss = dense.distill_loss(scores, cols, values)
    dense.adjust_scores(scores.detach(), bias=torch.ones(50, device="cuda"), out=scores.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name, device):
    """An operand with a tangent: the result would have none, a derivative of 0."""
    import torch.autograd.forward_ad as fwd
    fn, operands = small(device)[name]
    for which, t in operands.items():
        with fwd.dual_level():
            dual = fwd.make_dual(t.clone(), torch.ones_like(t))
            with pytest.raises(RuntimeError, match="forward-mode"):
                fn(**{**operands, which: dual})
    if device == "cuda":                                # a level that these operands are not part of is nobody's business
        with fwd.dual_level():
            fwd.make_dual(torch.ones(2), torch.ones(2))
            fn(**operands)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", CALLS)
def test_traces_are_refused(name, device):
    """A recorded graph would hold the output's allocation and nothing else."""
    from torch.fx.experimental.proxy_tensor import make_fx
    fn, operands = small(device)[name]
    fn_of = lambda *ts: fn(**dict(zip(operands, ts)))  # noqa: E731
    for kw in ({}, {"pre_dispatch": True}, {"tracing_mode": "fake"}):
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(fn_of, **kw)(*operands.values())
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(fn_of, tuple(operands.values()))
    if device == "cuda":
        fn(**operands)


@gpu
def test_compiled_programs():
    """torch.compile leaves the calls outside its graphs: the results are those of the eager program, gradients too."""
    cols, values = torch.tensor([[0, 1], [5, 2]], device="cuda"), torch.randn(2, 2, device="cuda")
    ids, ptr = torch.tensor([0, 3, 1], device="cuda"), torch.tensor([0, 2, 3], device="cuda")

    def program(table, weight):
        scores = torch.relu(dense.embed_rows(table, ids, ptr) @ weight) + 1.0
        loss = dense.distill_loss(scores, cols, values)
        return loss.sum(), dense.adjust_scores((scores * 2.0).detach(), bias=weight[0].detach())

    results = []
    for f in (program, torch.compile(program, backend="eager")):
        gen = torch.Generator(device="cuda").manual_seed(1)
        table, weight = (torch.randn(s, generator=gen, device="cuda").requires_grad_() for s in ((4, 6), (6, 9)))
        loss, scores = f(table, weight)
        loss.backward()
        results.append((loss.detach(), scores, table.grad, weight.grad))
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ---- bags beyond the launch of the column cut ------------------------------------------------------------------------------------

@gpu
def test_bags_more_than_the_column_cut_can_launch():
    """2^23 and more bags of a large table of rows of 1 KB: cut by columns they would need more threads than a launch has."""
    n, vocab, dim = 2**23 + 5, 100_000, 512
    gen = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randn(vocab, dim, generator=gen, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, vocab, (vocab + 1,), generator=gen, device="cuda", dtype=torch.int32)
    at = torch.arange(vocab + 1, device="cuda") * 83                                # rows with an entry, the last one among them
    at[-1] = n - 1
    indptr = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    indptr[at + 1] = 1
    indptr = torch.cumsum(indptr, 0, dtype=torch.int32)
    out = dense.embed_rows(table, ids, indptr)
    assert torch.equal(out[at], table[ids.long()])                                 # bags of one entry: the row itself
    filled = sum(int((part.view(torch.int16) != 0).any(1).sum()) for part in out.split(2**20))
    assert filled == vocab + 1


def embed_refusal(symbol="sp_embed_rows", **fields):
    """What the C entry says, without a device, to a call of these sizes: "" where it would launch."""
    import ctypes as C

    from similaripy_amd import _abi
    a = _abi.SpEmbedArgs()
    a.struct_size = C.sizeof(a)
    a.src = a.out = a.indices = a.workspace = 1 << 20
    a.workspace_bytes, a.scale = 1 << 60, 1.0
    for name, value in fields.items():
        setattr(a, name, value)
    rc = getattr(_abi.load(), symbol)(C.byref(a))
    assert rc in (-1, -2)                               # refused, or no device
    return _abi.last_error() if rc == -1 else ""


no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the calls name memory that is not there: only without a device")


@no_device
@pytest.mark.parametrize("dim", [512, 1024, 4096, 8192, 768, 1792, 2304])
def test_launch_limits_of_bags(dim):
    """Bags of bf16 rows: a wave for every slab of 1 KB whatever the column cut of large tables would need."""
    slabs = -(-dim // 512)
    limit = 4 * ((2**32 - 1) // 256 // slabs)           # four bags and one slab are a workgroup of 256 threads
    size = dict(dtype=1, out_dtype=1, n_vocab=100_000, dim=dim, ld_src=dim, ld_out=dim, nnz=200_000, indptr=1 << 20)
    for n in (1, 8192, 8193, 2**23 - 4, 2**23 - 3, 2**23, 2**24 + 1, limit):
        assert n > limit or embed_refusal(n_rows=n, **size) == ""
    for n in (limit + 1, 2**27):
        assert "too many rows" in embed_refusal(n_rows=n, **size)
    assert embed_refusal(n_rows=2**27, **{**size, "n_vocab": 0}) == ""


@no_device
@pytest.mark.parametrize("dtype,dim,lanes", [(0, 3, 8), (0, 32, 8), (0, 33, 16), (1, 128, 16), (1, 512, 64), (0, 256, 64), (0, 1000, 256)])
def test_launch_limits_of_lookups(dtype, dim, lanes):
    """A row of a lookup has 8 .. 64 lanes for every KB of it."""
    limit = (2**32 - 1) // 256 * 256 // lanes
    size = dict(dtype=dtype, out_dtype=dtype, n_vocab=100_000, dim=dim, ld_src=dim, ld_out=dim)
    assert embed_refusal(n_rows=limit, nnz=limit, **size) == ""
    assert "too many rows" in embed_refusal(n_rows=limit + 1, nnz=limit + 1, **size)


@no_device
@pytest.mark.parametrize("dtype", [0, 1])
def test_launch_limits_of_gradients(dtype):
    """Refused before anything is sorted or cleared: rows so wide that the sums, or the unsorted form, have more workgroups than a launch."""
    wide = 256 if dtype == 0 else 512                   # columns of a slab
    size = dict(dtype=dtype, out_dtype=dtype)
    for slabs, n, vocab, fits in ((4095, 102_400, 3, True), (4096, 102_400, 3, False), (2**14, 102_400, 3, False),          # 4096 chunks
                                  (16, 1000, 2**31 - 2, False), (15, 1000, 2**31 - 2, True), (2**20, 5, 15, True), (2**20, 5, 16, False)):
        dim = slabs * wide
        said = embed_refusal("sp_embed_rows_grad", n_rows=n, nnz=n, n_vocab=vocab, dim=dim, ld_src=dim, ld_out=dim, **size)
        assert said == "" if fits else "too many" in said, (slabs, n, vocab, said)


# ---- numbers -----------------------------------------------------------------------------------------------------------------------

@gpu
def test_numbers_on_the_device():
    """A parameter of no dimensions is read by the kernel: no wait for the device, a captured call follows its value."""
    z = torch.randn(3, 40, device="cuda")
    h = (torch.tensor([0, 2, 3, 3], device="cuda"), torch.tensor([4, 4, 9], device="cuda"))
    want = dense.adjust_scores(z, history=h, repetition=1.5, presence=0.25, frequency=2.0)
    p = [torch.tensor(x, device="cuda", dtype=t) for x, t in ((1.5, torch.float32), (0.25, torch.bfloat16), (2, torch.int64))]
    call = lambda: dense.adjust_scores(z, history=h, repetition=p[0], presence=p[1], frequency=p[2])  # noqa: E731
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        got = call()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(got, want)
    assert torch.equal(dense.adjust_scores(z, history=h, repetition=p[0].cpu(), presence=p[1].cpu(), frequency=p[2].cpu()), want)


@gpu
def test_numbers_on_the_device_captured():
    z = torch.randn(3, 40, device="cuda")
    h = (torch.tensor([0, 2, 3, 3], device="cuda"), torch.tensor([4, 4, 9], device="cuda"))
    p = [torch.tensor(x, device="cuda") for x in (1.5, 0.25, 2.0)]
    call = lambda: dense.adjust_scores(z, history=h, repetition=p[0], presence=p[1], frequency=p[2])  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = call()
    for x in (1.25, 2.0, 3.0):
        for t in p:
            t.fill_(x)
        g.replay()
        assert torch.equal(res, dense.adjust_scores(z, history=h, repetition=x, presence=x, frequency=x))
        torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_numbers_that_require_a_gradient(device):
    """scale, temperature, repetition, presence and frequency have no gradient: one that asks for it is refused, not read."""
    z = torch.randn(3, 40, device="cuda")
    ids = torch.tensor([0, 1], device="cuda")
    h = (torch.tensor([0, 2, 3, 3], device="cuda"), torch.tensor([4, 4, 9], device="cuda"))
    cols, values, stats = torch.tensor([[0, 1]] * 3, device="cuda"), torch.ones(3, 2, device="cuda"), torch.ones(3, 2, device="cuda")
    x = torch.tensor(1.5, device=device, requires_grad=True)
    for name, call in (("scale", lambda: dense.embed_rows(z, ids, scale=x)), ("scale", lambda: dense.embed_rows_grad(z[:2], ids, 3, scale=x)),
                       ("repetition", lambda: dense.adjust_scores(z, history=h, repetition=x)), ("presence", lambda: dense.adjust_scores(z, history=h, presence=x)),
                       ("frequency", lambda: dense.adjust_scores(z, history=h, frequency=x)),
                       ("temperature", lambda: dense.distill_loss(z, cols, values, temperature=x)),
                       ("temperature", lambda: dense.distill_loss(z.clone().requires_grad_(), cols, values, temperature=x)),
                       ("temperature", lambda: dense.distill_grad(z, stats, cols, values, temperature=x)),
                       ("temperature", lambda: dense.distill_loss_grad(z, cols, values, temperature=x))):
        with pytest.raises(ValueError, match=f"{name} has no gradient here"):
            call()
        with torch.no_grad():
            call()


@gpu
def test_statistics_of_another_layout():
    """Row statistics are pairs: [2, n] holds as many elements and is something else."""
    z = torch.randn(5, 40, device="cuda")
    cols, values = torch.tensor([[0, 1]] * 5, device="cuda"), torch.randn(5, 2, device="cuda")
    _, stats = dense.distill_loss(z, cols, values, return_stats=True)
    want = dense.distill_grad(z, stats, cols, values)
    for wrong in (stats.T, stats.T.contiguous(), stats.reshape(1, 5, 2), stats[:4]):
        with pytest.raises(ValueError, match="stats must"):
            dense.distill_grad(z, wrong, cols, values)
    assert torch.equal(dense.distill_grad(z, stats.reshape(-1), cols, values), want)
    assert torch.equal(dense.distill_grad(z, torch.stack([stats, stats], 2)[:, :, 0], cols, values), want)      # strided


# ---- outputs beside inputs ---------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_outputs_in_the_columns_beside_their_inputs(dtype):
    """Rows of one store: the output's columns lie beside the input's, before or behind them, one row further as well."""
    rng = np.random.default_rng(0)
    n, v = 6, 37
    store = torch.from_numpy(rng.standard_normal((n + 1, 3 * v))).to(dtype).cuda()
    keep = store.clone()
    bias = torch.from_numpy(rng.standard_normal(v)).to(dtype).cuda()
    cols, values = torch.tensor([[1, 5]] * n, device="cuda"), torch.randn(n, 2, device="cuda")
    ids = torch.arange(n, device="cuda")
    src = store[:n, v:2 * v]
    for out in (store[:n, :v], store[:n, 2 * v:], store[1:, :v], store[1:, 2 * v:]):
        assert torch.equal(dense.adjust_scores(src, bias=bias, out=out), dense.adjust_scores(src.clone(), bias=bias))
        assert torch.equal(dense.distill_loss_grad(src, cols, values, out=out)[1], dense.distill_loss_grad(src.clone(), cols, values)[1])
        assert torch.equal(dense.embed_rows(src, ids, out=out), src)
        assert torch.equal(dense.embed_rows_grad(src, ids, n, out=out), src)
        assert torch.equal(src, keep[:n, v:2 * v])
    one = store[2:3, :v]                                                           # one row between the rows of the other
    assert torch.equal(dense.embed_rows(src, ids[3:4], out=one), src[3:4])
    assert torch.equal(dense.adjust_scores(store[2:3, v:2 * v], bias=store[2, :v]), dense.adjust_scores(src[2:3].clone(), bias=store[2, :v].clone()))
    for out in (store[:n, 1:v + 1], store[:n, 2 * v - 1:3 * v - 1], store[1:, v:2 * v], store[1:, v + 1:2 * v + 1], store[n - 1:n, v - 1:2 * v - 1]):
        with pytest.raises(ValueError, match="shares memory"):
            if out.shape[0] == 1:
                dense.embed_rows(src, ids[:1], out=out)
            else:
                dense.adjust_scores(src, out=out)
    wide = torch.zeros(4 * n, v, dtype=dtype, device="cuda")                       # other distances between rows: only apart altogether
    with pytest.raises(ValueError, match="shares memory"):
        dense.adjust_scores(wide[:2 * n:2], out=wide[1:n + 1])
    dense.adjust_scores(wide[:2 * n:2], out=wide[2 * n:3 * n])


@gpu
def test_outputs_over_any_operand_are_refused():
    """Kernels read lists, weights and statistics while they write: an output over any of them is refused."""
    n, v = 4, 64
    raw = torch.zeros(4096, dtype=torch.float32, device="cuda")
    out = raw[:n * v].view(n, v)
    over = lambda numel, dtype=torch.float32: raw[100:100 + numel * (2 if dtype == torch.int64 else 1)].view(dtype)  # noqa: E731
    z, ids, ptr = torch.randn(n, v, device="cuda"), torch.tensor([0, 1, 2, 3], device="cuda"), torch.tensor([0, 1, 2, 3, 4], device="cuda")
    cols, values = torch.zeros(n, 2, dtype=torch.int64, device="cuda"), torch.ones(n, 2, device="cuda")
    stats = torch.ones(n, 2, device="cuda")
    i64 = torch.int64
    pattern = (ptr, ids)
    for call in (
        lambda: dense.embed_rows(z, over(4, i64), out=out), lambda: dense.embed_rows(z, ids, over(5, i64), out=out), lambda: dense.embed_rows(z, ids, ptr, over(4), out=out),
        lambda: dense.embed_rows_grad(z, over(4, i64), n, out=out), lambda: dense.embed_rows_grad(z, ids, n, over(5, i64), out=out),
        lambda: dense.embed_rows_grad(z, ids, n, ptr, over(4), out=out),
        lambda: dense.adjust_scores(z, targets=over(4, i64), out=out), lambda: dense.adjust_scores(z, allowed=over(2, torch.int32), out=out),
        lambda: dense.adjust_scores(z, filter_cols=(over(5, i64), ids), out=out), lambda: dense.adjust_scores(z, target_cols=(ptr, over(4, i64)), out=out),
        lambda: dense.adjust_scores(z, history=(ptr, over(4, i64)), out=out), lambda: dense.adjust_scores(z, history=pattern, repetition=over(4), out=out),
        lambda: dense.adjust_scores(z, history=pattern, presence=over(4), out=out), lambda: dense.adjust_scores(z, history=pattern, frequency=over(4), out=out),
        lambda: dense.distill_grad(z, over(8).view(n, 2), cols, values, out=out), lambda: dense.distill_grad(z, stats, over(8, i64), values, out=out),
        lambda: dense.distill_grad(z, stats, cols, over(8), out=out), lambda: dense.distill_grad(z, stats, cols, values, over(4, torch.int32), out=out),
        lambda: dense.distill_grad(z, stats, cols, values, grad_loss=over(4), out=out), lambda: dense.distill_grad(z, stats, cols, values, teacher_lse=over(4), out=out),
        lambda: dense.distill_loss_grad(z, over(8, i64), values, out=out), lambda: dense.distill_loss_grad(z, cols, over(8), out=out),
        lambda: dense.distill_loss_grad(z, cols, values, over(4, torch.int32), out=out), lambda: dense.distill_loss_grad(z, cols, values, grad_loss=over(4), out=out),
    ):
        with pytest.raises(ValueError, match="out shares memory"):
            call()


# ---- numbers at the ends of float32 --------------------------------------------------------------------------------------------

@gpu
def test_repetition_that_is_0_in_float32():
    z = torch.ones(1, 4, device="cuda")
    h = (torch.tensor([0, 1], device="cuda"), torch.tensor([2], device="cuda"))
    with pytest.raises(ValueError, match="repetition must be positive"):
        dense.adjust_scores(z, history=h, repetition=1e-46)
    assert dense.adjust_scores(z, history=h, repetition=2.0 ** -100)[0, 2].item() == 2.0 ** 100


def test_c_repetition_must_be_positive():
    """A history with a penalty but repetition_all left at 0 divides by 0."""
    import ctypes as C

    from similaripy_amd import _abi
    a = _abi.SpAdjustArgs()
    a.struct_size = C.sizeof(a)
    a.n_rows, a.n_cols, a.ld_scores, a.ld_out, a.device = 1, 4, 4, 4, 1 << 20      # (no such device: nothing is launched)
    a.scores = a.out = a.history.indptr = a.history.indices = 64
    a.history.n_rows = a.history.nnz = 1
    a.presence_all = 1.0
    for r in (0.0, -1.0, math.nan):
        a.repetition_all = r
        assert _abi.load().sp_adjust_scores(C.byref(a)) == -1 and "repetition" in _abi.last_error()
    a.repetition_all = 1.0
    assert _abi.load().sp_adjust_scores(C.byref(a)) < 0 and "repetition" not in _abi.last_error()


@gpu
@pytest.mark.parametrize("tau", [1e-25, 1e-21, 1e19, 1e21, 1e25])
def test_distill_temperatures_whose_square_leaves_float32(tau):
    """tau^2 is 0 or inf there, the loss is not: it is near tau (max - score) for small tau, and 0 of an empty list or for p = q."""
    z = torch.tensor([[3.0, 1.0, -2.0, 0.5], [1.0, 2.0, 4.0, 8.0]], device="cuda")
    cols, values = torch.tensor([[1, 2], [0, 1]], device="cuda"), torch.tensor([[5.0, 1.0], [1.0, 3.0]], device="cuda")
    counts = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    loss, stats = dense.distill_loss(z, cols, values, counts, temperature=tau, return_stats=True)
    one, grad = dense.distill_loss_grad(z, cols, values, counts, temperature=tau)
    assert torch.equal(loss, one) and loss[1].item() == 0.0 and (grad[1] == 0).all()
    if tau < 1:                                         # p is 1 at the list's best (column 1), q at the row's best
        assert abs(loss[0].item() - np.float32(tau) * 2.0) <= 1e-5 * tau
        assert (grad[0].double().cpu() - tau * torch.tensor([1.0, -1.0, 0.0, 0.0])).abs().max() <= 1e-6 * tau
    else:                                               # p is 1/2 twice, q 1/4: tau^2 log 2
        want = float(tau) ** 2 * math.log(2.0)
        assert loss[0].item() == math.inf if want > 3.5e38 else abs(loss[0].item() - want) <= 1e-5 * want
        assert (grad[0].double().cpu() / tau - torch.tensor([0.25, -0.25, -0.25, 0.25])).abs().max() <= 1e-6


@gpu
@pytest.mark.parametrize("n", [3, 300])
def test_distill_teacher_without_mass(n):
    """A teacher whose scores are all -inf has a log-sum-exp of -inf too: its list has no mass, loss and gradient are 0."""
    z = torch.randn(n, 40, device="cuda")
    cols, values = torch.tensor([[3, 7]] * n, device="cuda"), torch.ones(n, 2, device="cuda")
    lse = torch.full((n,), 2.0, device="cuda")
    values[1], lse[1] = -math.inf, -math.inf
    values[2, 0] = -math.inf
    loss, stats = dense.distill_loss(z, cols, values, teacher_lse=lse, return_stats=True)
    two = dense.distill_grad(z, stats, cols, values, teacher_lse=lse)
    one, grad = dense.distill_loss_grad(z, cols, values, teacher_lse=lse)
    assert torch.equal(one, loss) and loss[1].item() == 0.0 and (grad[1] == 0).all() and (two[1] == 0).all()
    assert loss.isfinite().all() and grad.isfinite().all() and grad[2, 7].item() < 0 < grad[2, 3].item()


# ---- refusals, each for its own reason -----------------------------------------------------------------------------------------

def refusals():
    """(call, exception, fragment of its message): every operand made for its call."""
    def Z(*shape, **kw):
        return torch.zeros(*(shape or (4, 6)), device="cuda", **kw)

    def I(*values, dtype=torch.int64):  # noqa: E743
        return torch.tensor(values, dtype=dtype, device="cuda")
    ids, i32 = I(0, 0, 0), I(0, 0, 0, 0, dtype=torch.int32)
    cols, vals = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), Z(4, 2)
    leaf = lambda *shape: Z(*shape).requires_grad_()  # noqa: E731
    E, G, A, L = dense.embed_rows, dense.embed_rows_grad, dense.adjust_scores, dense.distill_loss
    D, B = dense.distill_grad, dense.distill_loss_grad
    return [
        (lambda: E(Z().T, ids), ValueError, "table must have contiguous rows"), (lambda: E(Z(4), ids), ValueError, r"table must have 2 dimension"),
        (lambda: E([1], ids), TypeError, "table must be a torch.Tensor"), (lambda: E(Z().double(), ids), TypeError, "table must be float32, bfloat16 or float16"),
        (lambda: E(Z(), ids.float()), TypeError, "indices must be int32 or int64"), (lambda: E(Z(), [0]), TypeError, "indices must be a torch.Tensor"),
        (lambda: E(Z(), ids.cpu()), ValueError, "indices is on cpu"), (lambda: E(Z(), ids, i32), TypeError, "indptr must be int64"),
        (lambda: E(Z(), ids, None, Z(3)), ValueError, "data needs indptr"), (lambda: E(Z(), ids, I(0, 3), Z(2)), ValueError, "data must have 3 elements"),
        (lambda: E(Z(), ids, I(0, 3), Z(3).double()), TypeError, "data must be float32"), (lambda: E(Z(), ids, I(0, 3), leaf(3)), ValueError, "data has no gradient here"),
        (lambda: E(leaf(), ids, I(0, 3), leaf(3)), ValueError, "data has no gradient here"), (lambda: E(Z(), ids.reshape(3, 1), I(0, 3)), ValueError, "indices must have 1 dimension"),
        (lambda: E(Z(), ids, ids[:0]), ValueError, "indptr must have 1 dimension and at least one element"),
        (lambda: E(Z(), ids, out=[1]), TypeError, "out must be a torch.Tensor"), (lambda: E(Z(), ids, out=Z(3, 5)), ValueError, r"out must have shape \(3, 6\)"),
        (lambda: E(Z(), ids, out=Z(3, 6).half()), ValueError, "out must be torch.float32"), (lambda: (lambda t: E(t, ids, out=t[:3]))(Z()), ValueError, "shares memory"),
        (lambda: E(leaf(), ids, out=Z(3, 6)), ValueError, "builds no autograd graph"), (lambda: E(Z(), ids, out=leaf(3, 6)), ValueError, "out must not require a gradient"),
        (lambda: G([1], ids, 5), TypeError, "grad must be a torch.Tensor"), (lambda: G(Z(), ids, 5), ValueError, "grad has 4 rows, the indices make 3"),
        (lambda: G(Z(3, 6), ids, -1), ValueError, "n_vocab must not be negative"), (lambda: G(Z(3, 6), ids, 5, accumulate=True), ValueError, "accumulate needs out"),
        (lambda: G(Z(3, 6), ids, 5, dtype=torch.float16), ValueError, "the result must be torch.float32 or float32"),
        (lambda: G(leaf(3, 6), ids, 5), ValueError, "builds no autograd graph"), (lambda: G(Z(3, 6), ids, 5, out=Z(1, 6).expand(5, 6)), ValueError, "rows of out overlap"),
        (lambda: (lambda t: G(t[:3], ids, 4, out=t))(Z()), ValueError, "shares memory"),
        (lambda: A([1]), TypeError, "scores must be a torch.Tensor"), (lambda: A(leaf()), ValueError, "adjust_scores builds no autograd graph"),
        (lambda: A(Z(), targets=ids), ValueError, "targets must have 4 elements"), (lambda: A(Z(), targets=ids.float()), TypeError, "targets must be int32 or int64"),
        (lambda: A(Z(), history=i32), TypeError, r"history must be a pair \(indptr, indices\)"), (lambda: A(Z(), history=(i32, ids)), TypeError, "history must be int64"),
        (lambda: A(Z(), filter_cols=(ids[:0], ids)), ValueError, "filter_cols: indptr and indices"),
        (lambda: A(Z(), target_cols=(ids, ids.reshape(3, 1))), ValueError, "target_cols: indptr and indices"),
        (lambda: A(Z(), repetition=0.0), ValueError, "repetition must be positive"), (lambda: A(Z(), repetition=torch.tensor(0.0)), ValueError, "repetition must be positive"),
        (lambda: A(Z(), repetition=math.nan), ValueError, "repetition must be positive"), (lambda: A(Z(), repetition=Z(3)), ValueError, "repetition must have 4 elements"),
        (lambda: A(Z(), presence=Z(4).double()), TypeError, "presence must be float32"), (lambda: A(Z(), frequency=leaf(4)), ValueError, "frequency has no gradient here"),
        (lambda: A(Z(), bias=Z(5)), ValueError, r"bias must have shape \(6,\) or \(4, 6\)"), (lambda: A(Z(), bias=leaf(6)), ValueError, "builds no autograd graph"),
        (lambda: A(Z(), bias=Z(6, 4).T), ValueError, "bias must have contiguous rows"), (lambda: A(Z(), bias=Z(6).cpu()), ValueError, "bias must be on a HIP device"),
        (lambda: A(Z(), allowed=i32[:2]), ValueError, r"allowed must have shape \(1,\) or \(4, 1\)"), (lambda: A(Z(), allowed=ids[:1]), TypeError, "allowed must be int32"),
        (lambda: (lambda t: A(t[:3], out=t[1:]))(Z()), ValueError, "shares memory"), (lambda: A(Z(), out=Z(4, 7)), ValueError, r"out must be torch.float32 of shape \(4, 6\)"),
        (lambda: L([1], cols, vals), TypeError, "student must be a torch.Tensor"), (lambda: L(Z(), cols[:3], vals), ValueError, "cols must hold the same number of slots"),
        (lambda: L(Z(), cols.T, vals), ValueError, r"cols must have shape \(4, k\)"), (lambda: L(Z(), cols.float(), vals), TypeError, "cols must be int32 or int64"),
        (lambda: L(Z(), cols, vals[:3]), ValueError, r"values must have shape \(4, 2\)"), (lambda: L(Z(), cols, vals.T), ValueError, r"values must have shape \(4, 2\)"),
        (lambda: L(Z(), cols, vals.double()), TypeError, "values must be float32, bfloat16 or float16"), (lambda: L(Z(), cols, [1]), TypeError, "values must be a torch.Tensor"),
        (lambda: L(Z(), cols, vals.cpu()), ValueError, "values is on cpu"), (lambda: L(Z(), cols, leaf(4, 2)), ValueError, "values has no gradient here"),
        (lambda: L(leaf(), cols, leaf(4, 2)), ValueError, "values has no gradient here"), (lambda: L(Z(), cols, vals, ids), TypeError, "counts must be int32"),
        (lambda: L(Z(), cols, vals, i32[:3]), ValueError, "counts must have 4 elements"), (lambda: L(Z(), cols, vals, teacher_lse=Z(3)), ValueError, "teacher_lse must have 4 elements"),
        (lambda: L(leaf(), cols, vals, teacher_lse=leaf(4)), ValueError, "teacher_lse has no gradient here"),
        *((lambda t=t: L(Z(), cols, vals, temperature=t), ValueError, "temperature must be positive") for t in (0.0, -1.0, math.nan, math.inf)),
        (lambda: L(Z(), torch.zeros(4, 4097, dtype=torch.int32, device="cuda"), Z(4, 4097)), ValueError, "at most 4096"),
        (lambda: D(Z(), Z(4), cols, vals), ValueError, "stats must have 8 elements"), (lambda: D(leaf(), Z(4, 2), cols, vals), ValueError, "distill_grad builds no autograd graph"),
        (lambda: D(Z(), Z(4, 2), cols, vals, out=Z(4, 5)), ValueError, "out must be torch.float32 of shape"), (lambda: D(Z(), Z(4, 2).half(), cols, vals), TypeError, "stats must be float32"),
        (lambda: B(leaf(), cols, vals), ValueError, "distill_loss_grad builds no autograd graph"), (lambda: B(Z(), cols, vals, grad_loss=Z(3)), ValueError, "grad_loss must have 4 elements"),
        (lambda: B(Z(), cols, vals, out=Z(1, 6).expand(4, 6)), ValueError, "rows of out overlap"),
    ]


@gpu
def test_refusals_say_why():
    for i, (call, exception, message) in enumerate(refusals()):
        with pytest.raises(exception, match=message):
            call()
            raise AssertionError(f"call {i} went through: {message}")


# ---- score adjustment: histories at the limits of a segment's table and tiles -----------------------------------------------------

def long_history(rng, cols, distinct, entries, popular=0):
    """Ids of `distinct` of the columns, each at least once; one of them (and the column beside it) `popular` times more."""
    listed = rng.permutation(cols)[:distinct]
    more = entries - distinct - popular
    ids = np.concatenate([listed, np.full(popular, listed[0]), rng.choice(listed, more)])
    return rng.permutation(ids), np.bincount(ids, minlength=cols)


@gpu
@pytest.mark.parametrize("distinct,entries,popular", [(1024, 1024, 0), (1024, 1025, 1), (1024, 4000, 0), (1025, 1025, 0), (1025, 4000, 0), (1023, 70_000, 60_000),
                                                      (1025, 65_535, 64_510), (1025, 65_536, 64_511), (1500, 65_535, 60_000), (2048, 65_535, 0), (1500, 200_000, 150_000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_adjust_limits_of_the_table(dtype, distinct, entries, popular):
    """Rows of one segment of 2048 columns: as many distinct ids as the table takes and one more, histories that 16 bits count and one entry more,
    with a column that has nearly all of them between columns that have few."""
    rng = np.random.default_rng(distinct + entries)
    ids, count = long_history(rng, 2048, distinct, entries, popular)
    if popular:                                         # both halves of a word are counted
        a = ids[np.argmax(np.bincount(ids)[ids])]
        assert count[a] > popular
    count = torch.from_numpy(count)
    history = (torch.tensor([0, 0, entries], dtype=torch.int32, device="cuda"), torch.from_numpy(ids.astype(np.int32)).cuda())
    scores = torch.zeros(2, 2048, dtype=dtype, device="cuda")
    want = torch.stack([torch.zeros(2048), -count.float() / 16]).to(dtype)          # counts below 2^24: exact until the one rounding
    got = dense.adjust_scores(scores, history=history, frequency=1 / 16)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(dense.adjust_scores(scores, history=history, frequency=1 / 16, out=scores), got)


@gpu
@pytest.mark.parametrize("cols", [16_384, 40_001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adjust_tiles_of_wide_segments(dtype, cols):
    """Rows enough for segments of 14 336 and 16 384 columns: counts in two tiles of 16 bits and four of 32, in rows beside rows without a history."""
    rng = np.random.default_rng(cols)
    n = 2048
    kinds = [long_history(rng, cols, d, e, p) for d, e, p in ((cols * 5 // 16, 30_000, 0), (cols * 5 // 16, 65_535, 50_000), (cols * 5 // 16, 65_536, 50_000),
                                                             (cols, 300_000, 100_000), (700, 900, 0))]
    indptr = torch.from_numpy(np.cumsum([0] + [len(k[0]) for k in kinds])).to(torch.int32).cuda()
    history = (indptr, torch.from_numpy(np.concatenate([k[0] for k in kinds]).astype(np.int32)).cuda())
    targets = torch.full((n,), -1, dtype=torch.int32)
    at = torch.from_numpy(rng.permutation(n)[:40])
    targets[at] = torch.arange(40, dtype=torch.int32) % 5
    scores = torch.full((n, cols), 1.0, dtype=dtype, device="cuda")
    counts = torch.from_numpy(np.stack([k[1] for k in kinds])).float().cuda()
    # (2 - 1 on listed columns, then the count / 16; products and sums of small whole numbers over 16 are exact)
    listed = torch.where(counts > 0, 1.0 / 0.5 - (1.0 + counts / 16), 1.0).to(dtype)
    want = scores.clone()
    want[at.cuda()] = listed[(targets[at].long()).cuda()]
    kw = dict(targets=targets.cuda(), history=history, repetition=0.5, presence=1.0, frequency=1 / 16)
    got = dense.adjust_scores(scores, **kw)
    assert torch.equal(got, want)
    assert torch.equal(dense.adjust_scores(scores, out=scores, **kw), want)


# ---- types and strides that only the documentation names ----------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,k", [(3, 501, 20), (300, 9001, 130), (2, 120_001, 300)])
def test_distill_teachers_of_half_precision(dtype, vtype, n, v, k):
    """A teacher's values in 16 bits: the same as their float32 values, and the formula."""
    rng = np.random.default_rng(n + k)
    z = torch.from_numpy(rng.standard_normal((n, v)).astype(np.float32) * 3).to(dtype)
    cols = torch.from_numpy(np.stack([rng.permutation(v)[:k] for _ in range(n)]))
    values = torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32) * 2 + 3).to(vtype)
    counts = torch.from_numpy(rng.integers(0, k + 1, n).astype(np.int32))
    ref = distill_ref(z, cols, values, counts, 2.0, None, None)
    loss_b, grad_b = distill_bounds(z, cols, 2.0, ref, None, dtype)
    dev = (z.cuda(), cols.cuda(), values.cuda(), counts.cuda())
    loss, grad = dense.distill_loss_grad(*dev, temperature=2.0)
    check(loss, ref[0], loss_b, "loss")
    check(grad, ref[2], grad_b, "grad")
    wide = dense.distill_loss_grad(dev[0], dev[1], dev[2].float(), dev[3], temperature=2.0)
    assert torch.equal(loss, wide[0]) and torch.equal(grad, wide[1])
    one, stats = dense.distill_loss(*dev, temperature=2.0, return_stats=True)
    check(one, ref[0], loss_b, "loss alone")
    check(dense.distill_grad(dev[0], stats, *dev[1:], temperature=2.0), ref[2], grad_b, "grad alone")


@gpu
def test_strided_lists_and_parameters():
    """Every second element of a larger tensor, a column of a matrix, a row that stands for all: as their copies."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    i = lambda hi, *s: torch.randint(0, hi, s, generator=gen, device="cuda")  # noqa: E731
    every = lambda t: torch.stack([t, torch.full_like(t, 77)], -1)[..., 0]  # noqa: E731
    n, v, k = 5, 70, 6
    table, ids, ptr, w = r(v, 9), i(v, 40), torch.tensor([0, 3, 3, 20, 31, 40], device="cuda"), r(40)
    assert torch.equal(dense.embed_rows(table, every(ids), every(ptr), every(w)), dense.embed_rows(table, ids, ptr, w))
    look = i(v, 4, 6)
    assert torch.equal(dense.embed_rows(table, look.T), table[look.T])
    g = r(n, 9)
    assert torch.equal(dense.embed_rows_grad(g, every(ids), v, every(ptr), every(w)), dense.embed_rows_grad(g, ids, v, ptr, w))
    z, h = r(n, v), (torch.tensor([0, 2, 9, 9, 12, 15], device="cuda"), i(v, 15))
    rep, bias, bits = 1 + r(n).abs(), r(v), i(2**31 - 1, n, 3).int()
    want = dense.adjust_scores(z, targets=torch.arange(n, device="cuda"), history=h, repetition=rep, bias=bias, allowed=bits, filter_cols=h)
    pair = (every(h[0]), every(h[1]))
    assert torch.equal(dense.adjust_scores(z, targets=every(torch.arange(n, device="cuda")), history=pair, repetition=every(rep), bias=every(bias),
                                           allowed=every(bits), filter_cols=pair), want)
    assert torch.equal(dense.adjust_scores(z, bias=bias.expand(n, v)), dense.adjust_scores(z, bias=bias))
    cols, values, counts, lse, gl = i(v, n, k), r(n, k), torch.tensor([6, 0, 3, 1, 5], dtype=torch.int32, device="cuda"), r(n) + 4, r(n)
    want = dense.distill_loss_grad(z, cols, values, counts, grad_loss=gl, teacher_lse=lse)
    got = dense.distill_loss_grad(z, every(cols), every(values), every(counts), grad_loss=every(gl), teacher_lse=every(lse))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = dense.distill_loss_grad(z, cols, values, grad_loss=gl[:1].expand(n))
    assert torch.equal(one[1], dense.distill_loss_grad(z, cols, values, grad_loss=gl[:1].repeat(n))[1])


class Wrapped(torch.Tensor):
    """A tensor that keeps another one and has no memory of its own, as those of sharded or quantised models."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*[a.inner if isinstance(a, Wrapped) else a for a in args], **(kwargs or {}))


@gpu
def test_operands_without_memory():
    """Their pointer is 0, which says "not given" of an operand that may be left out: refused, as are those that may not."""
    z, ids, ptr, w = torch.randn(3, 40, device="cuda"), torch.tensor([0, 2, 1], device="cuda"), torch.tensor([0, 1, 3, 3], device="cuda"), torch.ones(3, device="cuda") * 2
    cols, values, counts = torch.tensor([[0, 1]] * 3, device="cuda"), torch.randn(3, 2, device="cuda"), torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")
    bits, row = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(40, device="cuda")
    W = Wrapped
    for call in (
        lambda: dense.embed_rows(z, ids, W(ptr)), lambda: dense.embed_rows(z, ids, ptr, W(w)), lambda: dense.embed_rows(W(z), ids), lambda: dense.embed_rows(z, W(ids)),
        lambda: dense.embed_rows_grad(z, ids, 3, ptr, W(w)), lambda: dense.embed_rows_grad(z, ids, 3, W(ptr), w), lambda: dense.embed_rows_grad(W(z), ids, 3),
        lambda: dense.adjust_scores(z, targets=W(ids)), lambda: dense.adjust_scores(z, bias=W(row)), lambda: dense.adjust_scores(z, allowed=W(bits)),
        lambda: dense.adjust_scores(z, filter_cols=(W(ptr), ids)), lambda: dense.adjust_scores(z, target_cols=(ptr, W(ids))),
        lambda: dense.adjust_scores(z, history=(ptr, ids), repetition=W(w)), lambda: dense.adjust_scores(z, history=(ptr, ids), presence=W(w)),
        lambda: dense.adjust_scores(z, history=(ptr, ids), frequency=W(w)), lambda: dense.adjust_scores(W(z)),
        lambda: dense.distill_loss(z, cols, values, W(counts)), lambda: dense.distill_loss(z, cols, values, teacher_lse=W(w)), lambda: dense.distill_loss(z, W(cols), values),
        lambda: dense.distill_loss(z, cols, W(values)), lambda: dense.distill_loss_grad(z, cols, values, grad_loss=W(w)), lambda: dense.distill_loss_grad(W(z), cols, values),
    ):
        with pytest.raises((TypeError, RuntimeError)):
            call()
    none = torch.zeros(0, device="cuda")                # empty operands have no memory either
    assert dense.adjust_scores(z[:0], history=(ptr, ids), repetition=none, frequency=none).shape == (0, 40)
    assert (dense.embed_rows(z, ids[:0], torch.zeros(3, dtype=torch.int64, device="cuda"), none) == 0).all()
