"""The softmax loss of pairs that are learnt (a loss near 0) keeps its digits.

Vectors of -1 and 1: every product is a whole number below 2^24, exact in float32 and bf16 whatever order it is summed in, so that what is
measured is the softmax alone.  A loss is log1p(exp(o - z)), o the logarithm over the other rows, z the target's logit: its relative error is
at most the absolute one of o - z.  That one, in float32's half steps: c = scale log2(e) is off by two of them, times at most 30, the distance
from z to the others' mean; the difference to the running maximum is rounded once, below 64 in base 2 (2^-25 * 64 * ln 2); the exponential is good
to 2^-22; 64 additions of positive terms in a lane and behind it; the result:  2^-23 * 30 + 1.3e-6 + 2^-22 + 2^-24 * 65 = 9e-6 if all of them
err by their most and the same way."""
import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
SLIP = 1e-5
SCALE = 30.0


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("opensearch_jvector_amd.ops")


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def learnt(torch, nq, n, d, dtype, sign=1.0, seed=0):
    """nq pairs with a cosine of 0.4 to 0.9 among n rows; the scale that makes a cosine of 1 a logit of SCALE."""
    rng = np.random.default_rng(1000 * nq + n + d + seed)
    v = rng.choice([-1.0, 1.0], (n, d))
    t = rng.permutation(n)[:nq]
    q = v[t] * sign
    for i in range(nq):
        q[i, rng.permutation(d)[:int(round(d * (0.05 + 0.25 * ((i * 7 + 3) % 10) / 10)))]] *= -1
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    return (torch.from_numpy(q).cuda().to(kind), torch.from_numpy(v).cuda().to(kind), torch.from_numpy(t.astype(np.int32)).cuda(), float(np.float32(sign * SCALE / d)))


def others(torch, q, v, t, scale):
    """Logits in float64, and o - z of each query, the target left out of o."""
    z = scale * (q.double() @ v.double().t())
    at = t.long()[:, None]
    hit = z.gather(1, at)[:, 0]
    return z, torch.logsumexp(z.scatter(1, at, float("-inf")), 1) - hit, hit


#       nq    n      d: every path and tile of the loss
PAIRS = [(1, 3770, 1000), (3, 3770, 1000), (4, 10000, 128), (2, 300, 96), (1, 2, 64), (4, 40000, 96), (70, 2000, 160), (60, 40000, 96), (90, 36000, 130), (130, 24000, 200),
         (300, 30011, 128), (257, 1500, 384), (2, 150001, 50)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d", PAIRS)
def test_a_loss_near_zero_keeps_its_digits(torch, ops, dtype, nq, n, d):
    q, v, t, scale = learnt(torch, nq, n, d, dtype)
    loss, lse = ops.softmax_loss(q, v, t, scale)
    z, apart, hit = others(torch, q, v, t, scale)
    want = torch.log1p(torch.exp(apart))
    assert want.min() < 0.02
    assert ((loss.double() - want).abs() <= SLIP * want).all(), ((loss.double() - want).abs() / want).max()
    # (the logits' own rounding: half a step of c, half a step of the result)
    assert ((lse.double() - (hit + want)).abs() <= 2.0 ** -23 * hit.abs() + SLIP * want + 2.0 ** -24 * (hit + want).abs()).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_negative_scale_and_several_queries_of_one_row(torch, ops, dtype):
    q, v, t, scale = learnt(torch, 3, 900, 200, dtype, sign=-1.0)
    q, t = torch.cat([q, q[:1], q[2:]]), torch.cat([t, t[:1], t[2:]])
    loss, _ = ops.softmax_loss(q, v, t, scale)
    want = torch.log1p(torch.exp(others(torch, q, v, t, scale)[1]))
    assert ((loss.double() - want).abs() <= SLIP * want).all() and torch.equal(loss[0], loss[3])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,d", [(300, 64), (3000, 700), (40000, 32)])
def test_what_a_loss_is_where_little_is_left(torch, ops, dtype, n, d):
    """One row alone; a scale of 0; what is not finite in the target's row, in another one, in the query."""
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(n)
    q, v = torch.randn((4, d), generator=g, device="cuda").to(kind), torch.randn((n, d), generator=g, device="cuda").to(kind)
    t = torch.tensor([0, 1, n - 1, -1], dtype=torch.int32, device="cuda")
    only = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, lse = ops.softmax_loss(q, v[:1], only, 1.0)
    z = (q.double() @ v[:1].double().t())[:, 0]
    # (a dot product of d terms, six times as many in float32)
    assert (loss == 0).all() and ((lse.double() - z).abs() <= (6 * d + 4) * 2.0 ** -23 * (q.double().abs() @ v[:1].double().abs().t())[:, 0]).all()
    loss, lse = ops.softmax_loss(q, v, t, 0.0)
    assert ((loss[:3] - np.log(n)).abs() <= 2.0 ** -20).all() and loss[3] == 0 and ((lse - np.log(n)).abs() <= 2.0 ** -20).all()
    for bad in (float("nan"), float("inf")):
        w = v.clone()
        w[1, 2] = bad
        loss, lse = ops.softmax_loss(q.abs(), w, t, 1.0)
        assert torch.isnan(loss[:3]).all() and loss[3] == 0 and torch.isnan(lse).all()
        x = q.clone()
        x[2, 1] = bad
        loss, lse = ops.softmax_loss(x, v.abs(), t, 1.0)
        assert torch.isnan(loss[2]) and torch.isnan(lse[2]) and torch.isfinite(loss[[0, 1, 3]]).all() and torch.isfinite(lse[[0, 1, 3]]).all()


def test_a_target_of_minus_infinity(torch, ops):
    """bf16 products are taken as they are: a target whose logit is -inf has probability 0 and an infinite loss, the others are as if it were absent."""
    v = torch.ones((40, 64), device="cuda", dtype=torch.bfloat16)
    v[5, 0] = float("-inf")
    q, t = torch.ones((2, 64), device="cuda", dtype=torch.bfloat16), torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    loss, lse = ops.softmax_loss(q, v, t, 0.125)
    assert loss[0] == float("inf") and abs(loss[1].item() - np.log(39)) <= 2.0 ** -20 and ((lse - (8 + np.log(39))).abs() <= 2.0 ** -20).all()


# ------------------------------------------------------------------------------------------------ gradients of learnt pairs
def gradients(torch, q, v, t, scale, w):
    """(dq, dv, reach of dq, reach of dv) in float64: g at the target from what its probability lacks to 1."""
    z, apart, hit = others(torch, q, v, t, scale)
    loss = torch.log1p(torch.exp(apart))
    g = torch.exp(z - (hit + loss)[:, None]).scatter(1, t.long()[:, None], torch.expm1(-loss)[:, None]) * (scale * w.double())[:, None]
    a, b = q.double(), v.double()
    return g @ b, g.t() @ a, g.abs() @ b.abs(), g.abs().t() @ a.abs()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d", PAIRS)
def test_a_learnt_pairs_gradient_keeps_its_digits(torch, ops, dtype, nq, n, d):
    """Row by row: an entry of g is off by SLIP (the target's), or by the lse's half step and the exponential's argument (the others': 2^-24 * 32 + SLIP); float32 g
    is held in three parts (2^-24), bf16 g in one (2^-8; the target's whole in dq); a sum of k terms in chains of k / 16 products of parts, six for
    float32, and so many half steps; the result is rounded once."""
    q, v, t, scale = learnt(torch, nq, n, d, dtype)
    w = torch.linspace(0.25, 1.0, nq, device="cuda")
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w, loss=loss)
    want_q, want_v, reach_q, reach_v = gradients(torch, q, v, t, scale, w)
    entry, last, parts = 2.0 ** -19 + SLIP + (2.0 ** -24 if dtype == "f32" else 2.0 ** -8), (2.0 ** -24 if dtype == "f32" else 2.0 ** -8), (6 if dtype == "f32" else 1)
    for got, want, reach, k in ((dq, want_q, reach_q, n), (dv, want_v, reach_v, nq)):
        off = (entry + (parts * k / 16 + 8) * 2.0 ** -24) * reach
        assert ((got.double() - want).abs() <= off + last * (want.abs() + off)).all(), ((got.double() - want).abs() / (off + last * want.abs())).max()
    # a row that is one query's target alone: its gradient is that query's, times the entry
    loss64 = torch.log1p(torch.exp(others(torch, q, v, t, scale)[1]))
    if nq == 1:
        own = (scale * w.double() * torch.expm1(-loss64))[:, None] * q.double()
        assert ((dv[t.long()].double() - own).abs() <= (2 * SLIP + 2 * last + (2.0 ** -8 if dtype == "bf16" else 0)) * own.abs()).all()
    one, none = ops.softmax_loss_grad(q, v, t, scale, lse, w, vectors_grad=False, loss=loss)
    assert none is None and torch.equal(one, dq)
    none, one = ops.softmax_loss_grad(q, v, t, scale, lse, w, queries_grad=False, loss=loss)
    assert none is None and torch.equal(one, dv)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_losses_of_queries_that_take_no_part_are_not_read(torch, ops, dtype):
    q, v, t, scale = learnt(torch, 9, 500, 96, dtype)
    t[[2, 5]] = torch.tensor([-1, 500], dtype=torch.int32, device="cuda")
    loss, lse = ops.softmax_loss(q, v, t, scale)
    want = ops.softmax_loss_grad(q, v, t, scale, lse, loss=loss)
    loss[[2, 5]] = torch.tensor([float("nan"), float("inf")], device="cuda")
    got = ops.softmax_loss_grad(q, v, t, scale, lse, loss=loss)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and (got[0][[2, 5]] == 0).all()
    with pytest.raises(ValueError):
        ops.softmax_loss_grad(q, v, t, scale, lse, loss=loss[:8])
    with pytest.raises(ValueError):
        ops.softmax_loss_grad(q, v, t, scale, lse, loss=loss.double())


def test_the_gradient_of_a_learnt_pair_is_the_losss_slope(torch, ops):
    """Against differences, at a loss of 1e-6, along the target's row and along another: components move by 2^-9, so that products stay exact.  A logit moves
    by r = SCALE 2^-9 at most; near 0 the loss is an exponential of the logits, so a central difference is off by (r^2 / 6) e^r of its reach, SCALE
    loss a unit, and the losses' own digits add SLIP e^r / r, the gradient's SLIP."""
    q, v, t, scale = learnt(torch, 1, 3770, 1000, "f32")
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, loss=loss)
    h, r = 2.0 ** -9, SCALE * 2.0 ** -9
    off = SCALE * loss.item() * (r * r / 6 * np.exp(r) + SLIP * np.exp(r) / r + 2 * SLIP)
    assert loss.item() < 1e-5
    for step in (v[t.long()], v[:1]):
        up, down = (ops.softmax_loss(q + sign * h * step, v, t, scale)[0].item() for sign in (1, -1))
        assert abs((up - down) / (2 * h) - (dq.double() * step.double()).sum().item()) <= off
    moved = [v.clone(), v.clone()]
    for x, sign in zip(moved, (1, -1)):
        x[t.long()] += sign * h * q
    up, down = (ops.softmax_loss(q, x, t, scale)[0].item() for x in moved)
    assert abs((up - down) / (2 * h) - (dv[t.long()].double() * q.double()).sum().item()) <= off
