"""The training and 8-bit scoring operators on the GPU against plain float64 implementations (tests/ops_support.py derives the bounds)."""
import importlib

import numpy as np
import pytest

import ops_support as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("opensearch_jvector_amd.ops")


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def dtype_of(torch, name):
    return torch.float32 if name == "f32" else torch.bfloat16


def matrix(torch, rng, n, d, dtype, pad=0, shift=0, unit=True):
    """[n][d] rows on the GPU, `pad` components apart, `shift` components into their storage; and their float64 values."""
    x = rng.standard_normal((n, d))
    if unit:
        x /= np.maximum(np.sqrt((x * x).sum(1, keepdims=True)), 1e-30)
    wide = torch.full((n * (d + pad) + shift + 1,), float("nan"), dtype=dtype_of(torch, dtype), device="cuda")
    rows = wide[shift:shift + n * (d + pad)].view(n, d + pad)[:, :d]
    rows.copy_(torch.from_numpy(x))
    return rows, rows.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ 8-bit rows
ENCODE = [(1, 1, 0, 0), (1, 128, 0, 0), (3, 129, 0, 0), (7, 127, 1, 0), (17, 384, 8, 4), (33, 1000, 0, 0), (5, 1536, 3, 1), (130, 64, 0, 0), (2, 4097, 0, 0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,d,pad,shift", ENCODE)
def test_encode_and_decode_bit_for_bit(torch, ops, dtype, n, d, pad, shift):
    rng = np.random.default_rng(n * 7 + d)
    x, x64 = matrix(torch, rng, n, d, dtype, pad, shift)
    x *= torch.exp2(torch.from_numpy(rng.integers(-30, 30, (n, 1)).astype(np.float32))).cuda().to(x.dtype)
    x64 = x.double().cpu().numpy()
    codes, scales = ops.encode_blocks(x)
    want_codes, want_scales = ref.encode(x64)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    values = ref.decode(want_codes, want_scales, d)
    assert np.array_equal(ops.decode_blocks(codes, scales, d).double().cpu().numpy(), values)   # 4 bits and a power of two: exact
    half = ops.decode_blocks(codes, scales, d, torch.bfloat16)
    assert np.array_equal(half.double().cpu().numpy(), values)                                   # in bf16 too


def test_encode_of_what_is_not_ordinary(torch, ops):
    """zeros, ties, both ends of the range, infinities and NaN, subnormal float32."""
    x = torch.zeros((12, 300), device="cuda")
    x[1, :4] = torch.tensor([448.0, 449.0, 464.0, -464.0])            # the block's scale doubles; ties between codes
    x[2, :3] = torch.tensor([448.0, 1.0625, 1.1875])                  # ties to the even code, both ways
    x[3, :2] = torch.tensor([float("inf"), 3.0])
    x[4, 5], x[4, 6], x[4, 130] = float("nan"), -2.0, float("-inf")
    x[5, :] = 3.4e38
    x[6, :3] = torch.tensor([1e-38, -1e-40, 2e-39])
    x[7, 299] = -7.0
    x[8, :2] = torch.tensor([-0.0, 1.0])
    x[9, :3] = torch.tensor([448.0, 2.0 ** -10, 1.5 * 2.0 ** -9])     # the smallest code, a tie to zero, a tie between subnormals
    x[10, 200] = 1e-45
    x[11, :] = torch.arange(300) - 150.0
    codes, scales = ops.encode_blocks(x)
    want_codes, want_scales = ref.encode(x.double().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    # float32 holds every such value but one: 3.4e38 / 2^120 = 255.8, its nearest code is 256, and 256 * 2^120 = 2^128 is float32's infinity
    with np.errstate(over="ignore"):
        values = ref.decode(want_codes, want_scales, 300).astype(np.float32)
    assert np.isinf(values[5]).all() and np.isfinite(values[[0, 1, 2, 6, 7, 8, 9, 10, 11]]).all()
    assert np.array_equal(ops.decode_blocks(codes, scales, 300).cpu().numpy(), values, equal_nan=True)
    # what is not finite stays visible in the scores, and only there
    scores = ops.score_blocks(codes, scales, codes[1:3].contiguous(), scales[1:3].contiguous(), 300).cpu().numpy()
    bad = np.isnan(scores).any(1)
    assert bad[3] and bad[4] and not bad[[0, 1, 2, 6, 7, 8, 9, 10, 11]].any()   # (row 5: infinities of both signs meet)


SCORE = [(1, 1, 1), (1, 300, 768), (5, 33, 128), (16, 129, 130), (33, 257, 1000), (64, 500, 64), (127, 128, 384), (129, 640, 100), (256, 1000, 768), (300, 77, 1536),
         (2, 1000, 4100), (513, 515, 257)]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d", SCORE)
def test_scores_of_encoded_rows(torch, ops, out, nq, n, d):
    rng = np.random.default_rng(nq + 3 * n + d)
    q, _ = matrix(torch, rng, nq, d, "f32", unit=False)
    v, _ = matrix(torch, rng, n, d, "f32", unit=False)
    v *= torch.exp2(torch.from_numpy(rng.integers(-20, 20, (n, 1)).astype(np.float32))).cuda()
    (qc, qs), (vc, vs) = ops.encode_blocks(q), ops.encode_blocks(v)
    a, b = (ref.decode(c.cpu().numpy(), s.cpu().numpy(), d) for c, s in ((qc, qs), (vc, vs)))
    want, reach = a @ b.T, np.abs(a) @ np.abs(b).T
    off = (d + 2) * 2.0 ** -23 * reach                                # d exact products summed in float32, however the unit rounds
    if out == "bf16":
        # the 8-bit unit adds 64 products at a time with a limited number of bits below the largest: 2^-11 of it by the entry's contract
        for k in range(0, d, 64):
            off = off + 2.0 ** -11 * np.max(np.abs(a[:, None, k:k + 64] * b[None, :, k:k + 64]), 2)
        off = off + 2.0 ** -8 * (np.abs(want) + off)
    got = ops.score_blocks(qc, qs, vc, vs, d, dtype_of(torch, out)).double().cpu().numpy()
    assert ref.far(got, want, off) <= 1


def test_a_run_of_rows_is_a_matrix_itself(torch, ops):
    rng = np.random.default_rng(5)
    v, _ = matrix(torch, rng, 400, 200, "f32")
    c, s = ops.encode_blocks(v)
    whole = ops.score_blocks(c[:9].contiguous(), s[:9].contiguous(), c, s, 200)
    part = ops.score_blocks(c[:9], s[:9], c[111:350], s[111:350], 200)
    assert torch.equal(whole[:, 111:350], part)


def test_scores_do_not_touch_what_lies_between_rows(torch, ops, pkg):
    b = pkg.binding
    rng = np.random.default_rng(6)
    v, _ = matrix(torch, rng, 150, 96, "f32")
    c, s = ops.encode_blocks(v)
    wide = torch.full((13, 200), 7.0, device="cuda")
    b.score_blocks_device(0, c.data_ptr(), s.data_ptr(), 12, c.data_ptr(), s.data_ptr(), 150, 96, b.DTYPE_F32, wide.data_ptr(), 200)
    assert torch.equal(wide[:12, :150], ops.score_blocks(c[:12], s[:12], c, s, 96))
    assert (wide[:12, 150:] == 7).all() and (wide[12] == 7).all()
    out = torch.full((151, 100), 7.0, device="cuda")
    b.decode_blocks_device(0, c.data_ptr(), s.data_ptr(), 150, 96, b.DTYPE_F32, out.data_ptr(), 100)
    assert torch.equal(out[:150, :96], ops.decode_blocks(c, s, 96)) and (out[:150, 96:] == 7).all() and (out[150] == 7).all()


# ------------------------------------------------------------------------------------------------ softmax loss
#      nq    n     d   pad shift scale
LOSS = [(1, 1, 1, 0, 0, 1.0), (1, 5, 3, 0, 0, 2.0), (3, 129, 64, 0, 0, 20.0), (2, 300, 17, 5, 1, 5.0), (129, 127, 65, 1, 3, 20.0), (64, 640, 128, 8, 0, 30.0),
        (130, 3000, 100, 0, 0, 10.0), (257, 1025, 384, 64, 8, 20.0), (31, 2000, 768, 0, 0, 20.0), (512, 260, 200, 0, 0, -3.0), (7, 1000, 1536, 0, 0, 50.0),
        (40, 130, 2, 1, 1, 3.0), (5, 70, 4, 0, 1, 3.0), (35, 77, 31, 0, 2, 9.0), (90, 261, 33, 6, 5, 9.0), (70, 300, 62, 3, 7, 9.0), (118, 18, 843, 24, 0, 10.0),
        (66, 520, 134, 2, 2, 12.0), (30, 1000, 72, 2, 2, 12.0), (100, 900, 8, 0, 0, 3.0), (61, 40, 200, 8, 6, 12.0), (28, 46, 1167, 0, 0, 12.0),
        (2, 3258, 1084, 0, 0, 12.0), (1, 1, 700, 3, 1, 1.0), (100, 2100, 519, 1, 1, -6.0), (33, 65, 2100, 8, 0, 20.0), (40, 200, 10, 0, 0, 9.0), (3, 1, 14, 2, 0, 2.0), (130, 700, 100, 0, 2, 10.0),
        (20, 129, 302, 4, 0, 15.0), (9, 64, 8, 0, 0, 3.0), (65, 2, 1022, 0, 0, 20.0)]


def loss_case(torch, nq, n, d, dtype, pad=0, shift=0, seed=0):
    rng = np.random.default_rng(nq * 31 + n * 7 + d + seed)
    v, v64 = matrix(torch, rng, n, d, dtype, pad, shift)
    q, _ = matrix(torch, rng, nq, d, dtype, pad, shift)
    t = rng.integers(0, max(n, 1), nq)
    near = rng.random((nq, 1)) * 0.9
    if n:
        q.copy_(torch.from_numpy(near * v64[t] + np.sqrt(1 - near * near) * q.double().cpu().numpy()))
    if nq > 4:
        t[1], t[3], t[4] = -1, n, t[0]          # none, out of range, a target shared
    if nq > 9:
        t[9] = -2 ** 31
    w = rng.random(nq).astype(np.float32)
    if nq > 6:
        w[6] = 0.0
    return q, v, torch.from_numpy(t.astype(np.int32)).cuda(), torch.from_numpy(w).cuda(), q.double().cpu().numpy(), v64, t, w.astype(np.float64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d,pad,shift,scale", LOSS)
def test_softmax_loss_and_gradients(torch, ops, dtype, nq, n, d, pad, shift, scale):
    q, v, t, w, q64, v64, t64, w64 = loss_case(torch, nq, n, d, dtype, pad, shift)
    want = ref.softmax(q64, v64, t64, scale, w64, dtype)
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w)
    assert dq.dtype == dv.dtype == q.dtype
    got = {"loss": loss, "lse": lse, "dq": dq, "dv": dv}
    off = {k: ref.far(got[k].double().cpu().numpy(), *want[k]) for k in got}
    assert max(off.values()) <= 1, off
    # one at a time gives the same bits, and so does a second call
    only_q, none = ops.softmax_loss_grad(q, v, t, scale, lse, w, vectors_grad=False)
    assert none is None and torch.equal(only_q, dq)
    none, only_v = ops.softmax_loss_grad(q, v, t, scale, lse, w, queries_grad=False)
    assert none is None and torch.equal(only_v, dv)
    again = ops.softmax_loss(q, v, t, scale)
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype,nq,n,d", [("bf16", 4096, 20011, 64), ("f32", 2500, 20011, 130), ("bf16", 1500, 70001, 64), ("f32", 64, 140001, 200),
                                          ("bf16", 4096, 140003, 64), ("f32", 4100, 45001, 20), ("f32", 3, 400001, 3), ("bf16", 5, 70001, 1001), ("bf16", 4096, 140003, 50), ("bf16", 4096, 140003, 51), ("bf16", 4096, 140003, 134)])
def test_softmax_over_several_pieces_of_the_rows(torch, ops, dtype, nq, n, d):
    """Sizes whose rows take several pieces: against a float64 computation on the GPU, with the bound's largest terms alone."""
    q, v, t, w, _, _, t64, _ = loss_case(torch, nq, n, d, dtype)
    scale = 20.0
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w)
    q64, v64 = q.double(), v.double()
    z = scale * (q64 @ v64.t())
    lse64 = torch.logsumexp(z, 1)
    known = (t >= 0) & (t < n)
    at = t.long().clamp(0, n - 1)
    rows = torch.arange(nq, device="cuda")
    # (terms + 2) 2^-23 of a logit's reach (rows have length about 1: scale), the logits' roundings, a sum of n terms
    de = (6 * d + 2) * 2.0 ** -23 * scale * 1.1 + 8 * 2.0 ** -24 * 2 * scale + n * 2.0 ** -24
    assert (lse - lse64).abs().max().item() <= de
    assert (loss - torch.where(known, lse64 - z[rows, at], torch.zeros_like(lse64))).abs().max().item() <= 2 * de
    g = torch.exp(z - lse64[:, None])
    g[rows, at] -= 1
    g *= (known * w * scale).double()[:, None]
    r = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -23
    for got, a, b, k in ((dq, g, v64, n), (dv, g.t(), q64, nq)):
        want, reach = a @ b, a.abs() @ b.abs()
        off = (r + 4 * de + 6 * k * 2.0 ** -23) * reach + 2 * ref.half_step(dtype) * want.abs()
        assert ((got.double() - want).abs() <= off + 1e-30).all()


def test_gradients_are_the_losses_slopes(torch, ops):
    """Against differences: the loss at vectors moved along a random direction, in float32 (step 2^-6: the third derivative's share is
    scale^3 step^2 / 6 of the direction's, the losses' rounding 2^-20 / step)."""
    q, v, t, w, *_ = loss_case(torch, 40, 500, 48, "f32")
    scale, h = 2.0, 2.0 ** -6
    _, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x, grad, move in ((q, dq, lambda s: (q + s, v)), (v, dv, lambda s: (q, v + s))):
        step = torch.randn(x.shape, generator=g, device="cuda")
        step /= step.norm(dim=1, keepdim=True)
        up, down = (float((w.double() * ops.softmax_loss(*move(sign * h * step), t, scale)[0].double()).sum()) for sign in (1, -1))
        slope, told = (up - down) / (2 * h), float((grad.double() * step.double()).sum())
        # every query's loss moves by at most 2 scale per unit, its third derivative by 8 (2 scale)^3 in all; weights are below 1
        assert abs(slope - told) <= 40 * (8 * scale ** 3 * h * h / 6 + 2.0 ** -19 * 8 / h)


def test_softmax_of_nothing(torch, ops):
    for dtype in (torch.float32, torch.bfloat16):
        q, v = torch.randn(5, 40, device="cuda").to(dtype), torch.randn(30, 40, device="cuda").to(dtype)
        t = torch.full((5,), -1, dtype=torch.int32, device="cuda")
        loss, lse = ops.softmax_loss(q, v, t, 1.0)
        assert (loss == 0).all() and torch.isfinite(lse).all()
        assert all((x == 0).all() for x in ops.softmax_loss_grad(q, v, t, 1.0, lse))
        loss, lse = ops.softmax_loss(q, v, None, 1.0)
        assert (loss == 0).all()
        assert all((x == 0).all() for x in ops.softmax_loss_grad(q, v, None, 1.0, lse))
        loss, lse = ops.softmax_loss(q, v[:0], t, 1.0)
        assert (loss == 0).all() and (lse == float("-inf")).all()
        dq, dv = ops.softmax_loss_grad(q, v[:0], t, 1.0, lse)
        assert (dq == 0).all() and dv.shape == (0, 40)
        loss, lse = ops.softmax_loss(q[:0], v, t[:0], 1.0)
        assert loss.shape == (0,)
        dq, dv = ops.softmax_loss_grad(q[:0], v, t[:0], 1.0, lse)
        assert dq.shape == (0, 40) and (dv == 0).all()
        # scale 0: every row is equally likely
        loss, lse = ops.softmax_loss(q, v, torch.arange(5, dtype=torch.int32, device="cuda"), 0.0)
        assert (lse - np.log(30)).abs().max() <= 2.0 ** -20
    assert ops.encode_blocks(torch.randn(0, 40, device="cuda"))[0].shape == (0, 128)
    c, s = ops.encode_blocks(torch.randn(3, 40, device="cuda"))
    assert ops.score_blocks(c[:0], s[:0], c, s, 40).shape == (0, 3) and ops.score_blocks(c, s, c[:0], s[:0], 40).shape == (3, 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_and_equal_logits(torch, ops, dtype):
    """Logits of some thousands (all but one probability 0), rows that are all alike, and logits whose largest is far below zero."""
    dt = dtype_of(torch, dtype)
    q, v = torch.zeros(4, 64, device="cuda", dtype=dt), torch.zeros(300, 64, device="cuda", dtype=dt)
    q[:, 0] = torch.tensor([64.0, -64.0, 0.0, 1.0])
    v[:, 0] = torch.arange(300).to(dt) / 4 if dtype == "f32" else torch.arange(300).to(dt)
    v[299, 0] = 300
    t = torch.tensor([299, 0, 7, 299], dtype=torch.int32, device="cuda")
    loss, lse = ops.softmax_loss(q, v, t, 1.0)
    z = q.double() @ v.double().t()
    want = torch.logsumexp(z, 1)
    assert (lse - want).abs().max().item() <= 2.0 ** -22 * z.abs().max().item() + 300 * 2.0 ** -24
    dq, dv = ops.softmax_loss_grad(q, v, t, 1.0, lse)
    assert torch.isfinite(dq.float()).all() and torch.isfinite(dv.float()).all()
    # the first query's answer has probability 1: what is left of its gradient is the lse's own error, times the rows' length
    assert abs(dq[0, 0].item()) <= 300 * 2.0 ** -21 * z.abs().max().item() and (dv[1:7] != 0).any()
    low = v.clone()
    low[:, 0] = -200
    loss, lse = ops.softmax_loss(q[:1], low, t[2:3], 1.0)
    assert abs(lse.item() - (-12800 + np.log(300))) <= 2.0 ** -22 * 12800 * 2 and abs(loss.item() - np.log(300)) <= 2.0 ** -22 * 12800 * 2


def test_a_row_that_is_not_finite_shows(torch, ops):
    q, v, t, w, *_ = loss_case(torch, 20, 200, 64, "f32")
    v = v.clone()
    v[77, 3] = float("nan")
    loss, lse = ops.softmax_loss(q, v, t, 5.0)
    assert torch.isnan(lse).all() and torch.isnan(loss[(t >= 0) & (t < 200)]).all() and (loss[1] == 0)
    v[77, 3] = 0.0
    q = q.clone()
    q[2, 0] = float("nan")
    loss, lse = ops.softmax_loss(q, v, t, 5.0)
    assert torch.isnan(lse[2]) and torch.isfinite(lse[torch.arange(20) != 2]).all()


@pytest.mark.parametrize("dtype,nq,n,d", [("f32", 40, 300, 700), ("f32", 100, 2000, 50), ("f32", 70, 40000, 96), ("f32", 150, 24000, 33), ("f32", 9, 70, 3), ("f32", 20, 300000, 2),
                                          ("bf16", 70, 500, 128), ("bf16", 70, 500, 100), ("bf16", 300, 30000, 192), ("bf16", 520, 17000, 72)])
def test_a_batch_padded_with_anything(torch, ops, dtype, nq, n, d):
    """Queries without a target take no part, whatever they, their lse and their weight hold: the same bits as with zeros."""
    q, v, t, w, *_ = loss_case(torch, nq, n, d, dtype)
    t[5::7] = -1
    t[nq - 2:] = torch.tensor([n, -7], dtype=torch.int32)
    dead = (t < 0) | (t >= n)
    q[dead] = 0
    want, lse = ops.softmax_loss(q, v, t, 9.0)
    grads = ops.softmax_loss_grad(q, v, t, 9.0, lse, w)
    garbage = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").to(q.dtype)
    q[dead] = garbage[torch.arange(int(dead.sum()), device="cuda") % 4][:, None].expand(-1, d).clone()
    got, lse2 = ops.softmax_loss(q, v, t, 9.0)
    assert torch.equal(got, want) and torch.equal(lse2[~dead], lse[~dead])
    lse2[dead], w[dead] = float("nan"), float("inf")
    dq, dv = ops.softmax_loss_grad(q, v, t, 9.0, lse2, w)
    assert torch.equal(dq, grads[0]) and torch.equal(dv, grads[1])
    assert (dq[dead] == 0).all() and torch.isfinite(dv.float()).all() and not (dv == 0).all()


def test_gradients_into_rows_that_lie_apart(torch, ops, pkg):
    b = pkg.binding
    q, v, t, w, *_ = loss_case(torch, 70, 333, 96, "bf16")
    _, lse = ops.softmax_loss(q, v, t, 8.0)
    dq, dv = ops.softmax_loss_grad(q, v, t, 8.0, lse, w)
    p = b.softmax_params(0, b.DTYPE_BF16, 70, 333, 96, 8.0, q.data_ptr(), q.stride(0), v.data_ptr(), v.stride(0), t.data_ptr())
    p.workspace_bytes = b.softmax_workspace(p, b.SOFTMAX_QUERY_GRAD | b.SOFTMAX_VECTOR_GRAD)
    ws = torch.empty(p.workspace_bytes + 64, dtype=torch.uint8, device="cuda").fill_(99)
    p.workspace = ws.data_ptr()
    oq, ov = torch.full((71, 101), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((334, 99), 5.0, dtype=torch.bfloat16, device="cuda")
    b.softmax_grad_device(p, lse.data_ptr(), w.data_ptr(), oq.data_ptr(), 101, ov.data_ptr(), 99)
    assert torch.equal(oq[:70, :96], dq) and torch.equal(ov[:333, :96], dv)
    assert (oq[:, 96:] == 5).all() and (oq[70] == 5).all() and (ov[:, 96:] == 5).all() and (ov[333] == 5).all()
    assert (ws[p.workspace_bytes:] == 99).all()


# ------------------------------------------------------------------------------------------------ streams and graphs
def step(torch, ops, q, v, t, w, scale=12.0):
    """The operators as they are used together: a training step of the rows, then 8-bit scores of the moved rows."""
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w)
    moved = v - 0.5 * dv
    codes, scales = ops.encode_blocks(moved)
    qc, qs = ops.encode_blocks(q)
    return loss, dq, dv, codes, scales, ops.score_blocks(qc, qs, codes, scales, v.shape[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_step_and_the_scores_after_it(torch, ops, dtype):
    q, v, t, w, *_ = loss_case(torch, 96, 2000, 160, dtype)
    loss, dq, dv, codes, scales, scores = step(torch, ops, q, v, t, w)
    moved = (v - 0.5 * dv).double().cpu().numpy()
    want_codes, want_scales = ref.encode(moved)
    assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), want_scales)
    a, b = ref.decode(*ref.encode(q.double().cpu().numpy()), 160), ref.decode(want_codes, want_scales, 160)
    assert ref.far(scores.double().cpu().numpy(), a @ b.T, 162 * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)) <= 1


def test_another_stream_and_two_at_once(torch, ops):
    cases = [loss_case(torch, 60, 3000, 128, "f32", seed=s)[:4] for s in (1, 2)]
    want = [step(torch, ops, *c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for s, c in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append([step(torch, ops, *c) for _ in range(3)])
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(x, y) for r in runs for x, y in zip(w, r))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_captured_step_replays(torch, ops, dtype):
    q, v, t, w, *_ = loss_case(torch, 50, 1500, 100, dtype)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(torch, ops, q, v, t, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(torch, ops, q, v, t, w)
    for k in range(5):
        v.mul_(1.0 + 0.125 * k)
        for x in out:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step(torch, ops, q, v, t, w)
        assert all(torch.equal(x, y) for x, y in zip(out, want)), k


def test_the_current_device_stays(torch, ops):
    before = torch.cuda.current_device()
    ops.encode_blocks(torch.randn(4, 8, device="cuda:0"))
    assert torch.cuda.current_device() == before


def test_refusals_of_the_torch_view(torch, ops, pkg):
    f, q, v = torch.float32, torch.randn(4, 32, device="cuda"), torch.randn(9, 32, device="cuda")
    t, c = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, 128, dtype=torch.uint8, device="cuda")
    s = torch.zeros(4, 1, dtype=torch.uint8, device="cuda")
    bad = [lambda: ops.encode_blocks(q.cpu()), lambda: ops.encode_blocks(q.half()), lambda: ops.encode_blocks(q[0]), lambda: ops.encode_blocks(q.t()),
           lambda: ops.decode_blocks(c, s, 129), lambda: ops.decode_blocks(c, s, 100, torch.float16), lambda: ops.decode_blocks(c[:, ::2], s, 64),
           lambda: ops.score_blocks(c, s, c, s[:3], 100), lambda: ops.score_blocks(c, s, c.cpu(), s.cpu(), 100),
           lambda: ops.softmax_loss(q, v.bfloat16(), t, 1.0), lambda: ops.softmax_loss(q, v[:, :31], t, 1.0), lambda: ops.softmax_loss(q, v, t.long(), 1.0),
           lambda: ops.softmax_loss(q, v, t[:3], 1.0), lambda: ops.softmax_loss_grad(q, v, t, 1.0, torch.zeros(3, device="cuda")),
           lambda: ops.softmax_loss_grad(q, v, t, 1.0, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda", dtype=torch.float64))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.softmax_loss(q, v[:1].expand(9, 32), t, 1.0), lambda: ops.softmax_loss(q, v, t, float("nan"))):
        with pytest.raises(pkg.binding.JvError) as e:
            call()
        assert e.value.code == pkg.binding.JV_EINVAL
    assert ops.softmax_loss_grad(q, v, t, 1.0, torch.zeros(4, device="cuda"), queries_grad=False, vectors_grad=False) == (None, None)


# ------------------------------------------------------------------------------------------------ the large tiles
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d", [(300, 33000, 200), (257, 24700, 1000), (2050, 6500, 128), (3100, 5000, 640), (70, 50001, 2200), (49153, 20, 64)])
def test_scores_on_the_large_tiles(torch, ops, out, nq, n, d):
    """Sizes that fill the chip with 256 x 256 tiles, none of them whole: scales of several windows, odd ends, rows that are not 16-B aligned."""
    g = torch.Generator(device="cuda").manual_seed(nq + n + d)
    q, v = (torch.randn((k, d), generator=g, device="cuda") * torch.exp2(torch.randint(-9, 9, (k, 1), generator=g, device="cuda")) for k in (nq, n))
    (qc, qs), (vc, vs) = ops.encode_blocks(q), ops.encode_blocks(v)
    a, b = (ops.decode_blocks(c, s, d).double() for c, s in ((qc, qs), (vc, vs)))
    want, off = a @ b.t(), (d + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if out == "bf16":
        for k in range(0, d, 64):   # 2^-11 of a group's largest product: at most of the product of the two largest components
            off += 2.0 ** -11 * a[:, k:k + 64].abs().amax(1)[:, None] * b[:, k:k + 64].abs().amax(1)[None]
        off += 2.0 ** -8 * (want.abs() + off)
    got = ops.score_blocks(qc, qs, vc, vs, d, dtype_of(torch, out))
    assert got.dtype == dtype_of(torch, out) and ((got.double() - want).abs() <= off).all()
    again = ops.score_blocks(qc, qs, vc, vs, d, dtype_of(torch, out))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype,nq,n,d,pad", [("bf16", 300, 30011, 200, 0), ("f32", 257, 26000, 70, 3), ("bf16", 1030, 10001, 384, 8), ("bf16", 80, 60000, 64, 0),
                                              ("f32", 600, 17000, 128, 0), ("f32", 600, 17000, 132, 0), ("bf16", 600, 17000, 128, 0), ("f32", 500, 25000, 129, 2), ("bf16", 400, 26000, 136, 2), ("bf16", 400, 26000, 8, 2), ("f32", 20, 40001, 70, 1), ("f32", 64, 33000, 3, 0),
                                              ("f32", 90, 36000, 130, 0), ("f32", 130, 24000, 100, 5), ("f32", 700, 9000, 36, 1),
                                              ("bf16", 3900, 3901, 200, 0), ("bf16", 2100, 500, 96, 0), ("bf16", 5000, 130, 70, 1), ("f32", 2100, 500, 96, 0), ("f32", 2500, 2600, 61, 2),
                                              ("f32", 5000, 130, 40, 0), ("bf16", 300, 30011, 100, 0), ("bf16", 700, 20000, 254, 2), ("bf16", 1000, 13001, 390, 0), ("bf16", 20000, 130, 24, 0)])
def test_softmax_on_the_large_tiles(torch, ops, dtype, nq, n, d, pad):
    q, v, t, w, _, _, t64, _ = loss_case(torch, nq, n, d, dtype, pad)
    scale = 15.0
    loss, lse = ops.softmax_loss(q, v, t, scale)
    z = scale * (q.double() @ v.double().t())
    lse64 = torch.logsumexp(z, 1)
    known = (t >= 0) & (t < n)
    at = t.long().clamp(0, n - 1)
    # (terms + 2) 2^-23 of a logit's reach (rows have length about 1: scale), the logits' roundings, a sum of n terms
    de = (6 * d + 2) * 2.0 ** -23 * scale * 1.1 + 8 * 2.0 ** -24 * 2 * scale + n * 2.0 ** -24
    assert (lse - lse64).abs().max().item() <= de
    assert (loss - torch.where(known, lse64 - z[torch.arange(nq, device="cuda"), at], torch.zeros_like(lse64))).abs().max().item() <= 2 * de
    p = torch.exp(z - lse64[:, None]) * (known * w * scale).double()[:, None]
    g = p.clone()
    g[torch.arange(nq, device="cuda"), at] -= (known * w * scale).double()
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w)
    r = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -23
    # An exponent that is off by de makes p, not g, off by that share: at a target with p near 1, g = p - 1 is near 0 and its error is still p de.
    for got, a, of, b, k in ((dq, g, p, v.double(), n), (dv, g.t(), p.t(), q.double(), nq)):
        want, reach = a @ b, a.abs() @ b.abs()
        assert ((got.double() - want).abs() <= (r + 6 * k * 2.0 ** -23) * reach + 4 * de * (of @ b.abs()) + 2 * ref.half_step(dtype) * want.abs() + 1e-30).all()


# ------------------------------------------------------------------------------------------------ offsets that pass 32 bits
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_lie_far_apart(torch, ops, dtype):
    """70 000 components from row to row, 4.9 G in all: the same bits as with the rows side by side."""
    q, v, t, w, *_ = loss_case(torch, 33, 70001, 24, dtype)
    wide = torch.empty(70001 * 70000, dtype=v.dtype, device="cuda")
    far = wide.view(70001, 70000)[:, 69976:]
    far.copy_(v)
    want, got = step(torch, ops, q, v, t, w), step(torch, ops, q, far, t, w)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_gradient_of_more_than_4_gib(torch, ops):
    n, d = 1200001, 1000
    g = torch.Generator(device="cuda").manual_seed(5)
    v = torch.randn((n, d), generator=g, device="cuda") / 32
    q, t = v[[3, n - 2, n // 2]] * 1.0, torch.tensor([3, n - 2, 9], dtype=torch.int32, device="cuda")
    loss, lse = ops.softmax_loss(q, v, t, 10.0)
    _, dv = ops.softmax_loss_grad(q, v, t, 10.0, lse, queries_grad=False)
    total = torch.zeros(3, dtype=torch.float64, device="cuda")
    for at in range(0, n, 100000):
        total += torch.exp(10.0 * (q.double() @ v[at:at + 100000].double().t())).sum(1)   # (|z| stays below 20)
    de = (6 * d + 2) * 2.0 ** -23 * 12 + n * 2.0 ** -24   # a logit's sum (its reach: below 12), the sum of n exponentials
    assert (lse - total.log()).abs().max().item() <= de
    for rows in (slice(0, 1000), slice(n // 2 - 500, n // 2 + 500), slice(n - 1000, n)):
        p = torch.exp(10.0 * (q.double() @ v[rows].double().t()) - total.log()[:, None])
        part = p.clone()
        for i in range(3):
            if rows.start <= int(t[i]) < rows.stop:
                part[i, int(t[i]) - rows.start] -= 1
        want = 10.0 * part.t() @ q.double()
        off = 10.0 * (4 * de * p.t() + 2.0 ** -20 * part.abs().t()) @ q.double().abs() + 2.0 ** -23 * want.abs()
        assert ((dv[rows].double() - want).abs() <= off + 1e-30).all()


def test_as_many_and_as_long_queries_as_few_tiles_take(torch, ops):
    """2^15 queries of 2^16 components against 16 rows: 8 GiB of queries, of their gradient and of their copy."""
    nq, n, d = 1 << 15, 16, 1 << 16
    g = torch.Generator(device="cuda").manual_seed(8)
    v = torch.randn((n, d), generator=g, device="cuda") / 256
    q = torch.empty((nq, d), device="cuda")
    for at in range(0, nq, 4096):
        q[at:at + 4096] = torch.randn((4096, d), generator=g, device="cuda") / 256
    t = (torch.arange(nq, device="cuda") % 17).int()   # (every 17th has none)
    loss, lse = ops.softmax_loss(q, v, t, 2.0)
    dq, dv = ops.softmax_loss_grad(q, v, t, 2.0, lse)
    want, reach = torch.zeros((n, d), dtype=torch.float64, device="cuda"), torch.zeros((n, d), dtype=torch.float64, device="cuda")
    # a dot product is 6 d / 16 additions of partial sums below 2^-5 (256 terms' root of 2^-16 each is 2^-8), half a step each, times the scale;
    # the exponentials and the logarithm of 16 of them: a few steps of 4
    de = 2 * 6 * d / 16 * 2.0 ** -24 * 2.0 ** -5 + 2.0 ** -20
    for at in range(0, nq, 2048):
        x = q[at:at + 2048].double()
        z = 2.0 * x @ v.double().t()
        assert (lse[at:at + 2048] - torch.logsumexp(z, 1)).abs().max().item() <= de
        p = torch.softmax(z, 1)
        p[torch.arange(2048, device="cuda"), t[at:at + 2048].long().clamp(max=15)] -= 1
        p *= 2.0 * (t[at:at + 2048] < 16).double()[:, None]
        want += p.t() @ x
        reach += p.abs().t() @ x.abs()
        if at % 8192 == 0:
            assert ((dq[at:at + 2048].double() - p @ v.double()).abs() <= 8 * de * (p.abs() @ v.double().abs())).all()
    assert ((dv.double() - want).abs() <= (8 * de + 6 * nq / 16 * 2.0 ** -24) * reach).all()


def test_codes_and_scores_of_more_than_4_gib(torch, ops):
    n, d = 4500001, 1000
    g = torch.Generator(device="cuda").manual_seed(6)
    v = torch.empty((n, d), dtype=torch.bfloat16, device="cuda")
    for at in range(0, n, 500000):
        v[at:at + 500000] = torch.randn((min(500000, n - at), d), generator=g, device="cuda")
    codes, scales = ops.encode_blocks(v)
    tail = slice(n - 1000, n)
    some, some_scales = ops.encode_blocks(v[tail].clone())
    assert torch.equal(codes[tail], some) and torch.equal(scales[tail], some_scales)
    assert torch.equal(ops.decode_blocks(codes, scales, d, torch.bfloat16)[tail], ops.decode_blocks(some, some_scales, d, torch.bfloat16))
    del v
    nq = 600   # 2.7 G scores
    got = ops.score_blocks(codes[:nq].contiguous(), scales[:nq].contiguous(), codes, scales, d)
    a, b = ops.decode_blocks(codes[:nq].contiguous(), scales[:nq].contiguous(), d).double(), ops.decode_blocks(some, some_scales, d).double()
    assert ((got[:, tail].double() - a @ b.t()).abs() <= (d + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t())).all()
