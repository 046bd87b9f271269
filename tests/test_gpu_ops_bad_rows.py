"""Rows that are not finite in the softmax loss's gradients: they reach the queries that have a target, and nothing else."""
import importlib

import numpy as np
import pytest

from ops_support import half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("opensearch_jvector_amd.ops")


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


#         float32: few tiles (one and several k ranges of dq, four waves a tile), planes of 32 to 128 queries; bf16: small tiles, large ones with and without
#         gradients on small ones, rows that are laid out (odd d), several pieces of g
SHAPES = [("f32", 5, 70, 30), ("f32", 40, 300, 700), ("f32", 33, 5000, 64), ("f32", 9, 70, 3), ("f32", 20, 45000, 64), ("f32", 90, 36000, 40), ("f32", 150, 24000, 33),
          ("bf16", 5, 70, 30), ("bf16", 70, 500, 100), ("bf16", 40, 700, 129), ("bf16", 300, 30000, 192), ("bf16", 520, 17000, 72), ("bf16", 300, 30000, 131),
          ("bf16", 4096, 140003, 64)]


def inputs(torch, dtype, nq, n, d):
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(nq + n + d)
    q, v = torch.randn((nq, d), generator=g, device="cuda").to(kind), torch.randn((n, d), generator=g, device="cuda").to(kind)
    return q, v, torch.randint(0, n, (nq,), generator=g, device="cuda").int(), torch.rand(nq, generator=g, device="cuda") + 0.5


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("dtype,nq,n,d", SHAPES)
def test_queries_without_a_target_beside_a_bad_row(torch, ops, dtype, nq, n, d, bad):
    q, v, t, w = inputs(torch, dtype, nq, n, d)
    t[1::3] = -1
    t[4] = n
    dead = (t < 0) | (t >= n)
    v[n - 1, d - 1] = v[n // 2, 0] = float(bad)
    with_loss, lse = ops.softmax_loss(q, v, t, 0.5)
    assert (with_loss[dead] == 0).all()
    for loss in (None, with_loss):
        dq, dv = ops.softmax_loss_grad(q, v, t, 0.5, lse, w, loss=loss)
        assert (dq[dead] == 0).all()
        # a logit that is NaN or +inf leaves no probabilities: its query's gradient and all rows' are NaN
        gone = ~torch.isfinite(lse) & ~dead
        assert torch.isnan(dq[gone].float()).all()
        if bad == "nan" or dtype == "f32":
            assert gone.sum() == (~dead).sum()
        if gone.any():
            assert torch.isnan(dv.float()).all()
    # none of them has one: no gradient at all, as with no targets
    t[:] = -1
    loss, lse = ops.softmax_loss(q, v, t, 0.5)
    dq, dv = ops.softmax_loss_grad(q, v, t, 0.5, lse, w, loss=loss)
    assert (loss == 0).all() and (dq == 0).all() and (dv == 0).all()
    for only in (dict(vectors_grad=False), dict(queries_grad=False)):
        assert all(x is None or (x == 0).all() for x in ops.softmax_loss_grad(q, v, t, 0.5, lse, w, **only))


@pytest.mark.parametrize("dtype,nq,n,d", SHAPES)
def test_a_weight_or_an_lse_that_is_not_finite_shows(torch, ops, dtype, nq, n, d):
    q, v, t, w = inputs(torch, dtype, nq, n, d)
    loss, lse = ops.softmax_loss(q, v, t, 0.5)
    for name in ("w", "lse"):
        x = {"w": w.clone(), "lse": lse.clone()}
        x[name][2] = float("nan")
        dq, dv = ops.softmax_loss_grad(q, v, t, 0.5, x["lse"], x["w"])
        assert torch.isnan(dq[2].float()).all() and torch.isfinite(dq[:2].float()).all() and torch.isfinite(dq[3:].float()).all()
        assert torch.isnan(dv.float()).all()
    w[2] = float("inf")
    dq, dv = ops.softmax_loss_grad(q, v, t, 0.5, lse, w)
    assert not torch.isfinite(dq[2].float()).any() and torch.isfinite(dq[:2].float()).all() and torch.isfinite(dq[3:].float()).all()
    assert not torch.isfinite(dv.float()).any()


def test_a_weight_of_zero_beside_a_bad_row(torch, ops):
    """A query that has a target takes part, whatever its weight: 0 * NaN is NaN."""
    for dtype in ("f32", "bf16"):
        q, v, t, w = inputs(torch, dtype, 6, 200, 64)
        w[:] = 0.0
        v[7, 7] = float("nan")
        loss, lse = ops.softmax_loss(q, v, t, 0.5)
        dq, dv = ops.softmax_loss_grad(q, v, t, 0.5, lse, w)
        assert torch.isnan(dq.float()).all() and torch.isnan(dv.float()).all()


def test_a_row_of_minus_infinite_logits_is_left_out(torch, ops):
    """bf16: its probability is 0, the other rows' gradients are as without it."""
    q, v, t, w = inputs(torch, "bf16", 12, 300, 64)
    q, t = q.abs(), t % 299
    t[3] = -1
    loss, lse = ops.softmax_loss(q, v[:299], t, 0.125)
    _, want = ops.softmax_loss_grad(q, v[:299], t, 0.125, lse, w, queries_grad=False, loss=loss)
    v[299, 5] = float("-inf")
    got_loss, got_lse = ops.softmax_loss(q, v, t, 0.125)
    assert ((got_lse - lse).abs() <= 2.0 ** -20 * lse.abs()).all()
    dq, dv = ops.softmax_loss_grad(q, v, t, 0.125, got_lse, w, loss=got_loss)
    # (one rounding of g and one of the result may fall the other way: half a step each, twice)
    assert (dv[299] == 0).all() and ((dv[:299].double() - want.double()).abs() <= 4 * half_step("bf16") * np.abs(want.abs().double().max().item())).all()
    assert (dq[3] == 0).all()


@pytest.mark.parametrize("dtype,nq,n,d", SHAPES)
def test_a_scale_of_zero_beside_an_infinite_product(torch, ops, dtype, nq, n, d):
    """0 times infinity is NaN, whatever its sign; no row is left out of the others' sum."""
    q, v, t, w = inputs(torch, dtype, nq, n, d)
    loss, lse = ops.softmax_loss(q, v, t, 0.0)
    assert ((lse - np.log(n)).abs() <= 2.0 ** -19).all() and ((loss - np.log(n)).abs() <= 2.0 ** -19).all()
    for bad in (float("inf"), -float("inf")):
        v[n // 2, 0] = bad
        loss, lse = ops.softmax_loss(q.abs() + 1, v, t, 0.0)
        assert torch.isnan(loss).all() and torch.isnan(lse).all()
