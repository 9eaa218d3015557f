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
