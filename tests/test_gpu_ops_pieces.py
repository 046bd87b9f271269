"""The softmax loss over rows that take several pieces, forward and backward, and over many rows: what a lost row, tile or piece would change.

Counted rows: row j is the unit vector of block j d / n, query i is a_i times ones, so that every logit of a query is scale a_i: exact, and the same.  Then each
term of the running sum is 1 and the sum a whole number (exact below 2^24 rows a lane), lse_i = scale a_i + log n, p = 1 / n, and with c_b the rows of block b
    loss_i = log n      dq_i[b] = w_i scale (c_b / n - [b is the target's])      dv_j = scale sum_i w_i a_i (1 / n - [j = t_i])
Bounds: log n and lse are rounded once, the join's partial sums are exact: three steps of |lse|.  p is exp of a difference of two such and off by 2^-19
of itself (|lse| below 32), float32 g by 2^-23 more, bf16 g by half a step; sums of k equal terms in float32 by k / 16 half steps at most; one rounding at the end."""
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


def pieces(b, dtype, nq, n, d, what, v, bytes_a_row):
    """At least how many pieces the rows of a call take: its workspace has no room for more than n / pieces of them."""
    p = b.softmax_params(0, dtype, nq, n, d, 1.0, 0, 0, v.data_ptr(), v.stride(0))
    return int(np.ceil(n * bytes_a_row / b.softmax_workspace(p, what | b.SOFTMAX_AS_THEY_LIE)))


def counted(torch, dtype, nq, n, d):
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    block = torch.arange(n, device="cuda") * d // n
    v = torch.zeros((n, d), dtype=kind, device="cuda")
    v[torch.arange(n, device="cuda"), block] = 1.0
    a = 2.0 ** (torch.arange(nq, device="cuda") % 3 - 1).double()
    t = (torch.arange(nq, device="cuda", dtype=torch.int64) * 7919 % n).int()
    t[nq // 2] = n - 1
    if nq > 4:
        t[3::5] = -1
    return v, a[:, None].expand(nq, d).to(kind).contiguous(), a, t, block


#         dtype   nq       n        d    pieces forward, backward (at least)
COUNTED = [("bf16", 5, 600001, 1001, 3, 1), ("bf16", 300, 400001, 1001, 4, 1), ("bf16", 300, 1200001, 1001, 8, 2), ("bf16", 4096, 500001, 64, 1, 4),
           ("bf16", 128, 9000001, 11, 8, 3), ("f32", 700, 600001, 20, 1, 3), ("f32", 64, 6000001, 3, 15, 3), ("bf16", 1 << 20, 513, 8, 1, 1), ("f32", 1 << 20, 513, 8, 1, 2),
           ("f32", 3, 1200001, 1000, 1, 1), ("bf16", 4096, 140003, 64, 1, 2), ("f32", 64, 140001, 200, 1, 1), ("f32", 300, 70001, 130, 1, 1), ("bf16", 64, 33000, 300, 1, 1)]


@pytest.mark.parametrize("dtype,nq,n,d,forward,backward", COUNTED)
def test_every_row_counts(torch, ops, pkg, dtype, nq, n, d, forward, backward):
    b = pkg.binding
    kind = b.DTYPE_F32 if dtype == "f32" else b.DTYPE_BF16
    v, q, a, t, block = counted(torch, dtype, nq, n, d)
    planes = 3 if dtype == "f32" else 1
    laid = (-(-d // 64) * 128 if d % 2 else 0) if dtype == "bf16" else (16 if d < 4 else 0)   # bytes of a row that is laid out
    if forward > 1:
        assert pieces(b, kind, nq, n, d, b.SOFTMAX_LOSS, v, laid) >= forward
    if backward > 1:
        assert pieces(b, kind, nq, n, d, b.SOFTMAX_QUERY_GRAD, v, laid + nq * planes * 2) >= backward
    scale = 0.75
    w = ((torch.arange(nq, device="cuda") % 7 + 1) / 8).float()
    loss, lse = ops.softmax_loss(q, v, t, scale)
    known, step = t >= 0, half_step(dtype)
    want = scale * a + np.log(n)
    assert ((lse.double() - want).abs() <= 3 * 2.0 ** -23 * want).all()
    assert ((loss.double() - known * np.log(n)).abs() <= 3 * 2.0 ** -23 * (np.log(n) + scale * a)).all()
    # outputs of NaN: what is not written shows
    p = b.softmax_params(0, kind, nq, n, d, scale, q.data_ptr(), d, v.data_ptr(), d, t.data_ptr())
    p.workspace_bytes = b.softmax_workspace(p, b.SOFTMAX_QUERY_GRAD | b.SOFTMAX_VECTOR_GRAD | b.SOFTMAX_AS_THEY_LIE)
    ws = torch.empty(p.workspace_bytes, dtype=torch.uint8, device="cuda").fill_(255)
    p.workspace = ws.data_ptr()
    dq, dv = torch.full_like(q, float("nan")), torch.full_like(v, float("nan"))
    b.softmax_grad_device(p, lse.data_ptr(), w.data_ptr(), dq.data_ptr(), d, dv.data_ptr(), d, 0, loss.data_ptr())
    del ws
    by = (known * w * scale).double()
    entry = 2.0 ** -19 + (step if dtype == "bf16" else 2.0 ** -23)
    count = torch.bincount(block, minlength=d).double()[None]
    for at in range(0, nq, 1 << 16):
        part = slice(at, at + (1 << 16))
        hit = torch.zeros((len(dq[part]), d), dtype=torch.float64, device="cuda")
        hit[torch.arange(len(hit), device="cuda"), block[t[part].long().clamp(min=0)]] = 1.0
        want, reach = by[part, None] * (count / n - hit), by[part, None] * (count / n + hit)
        off = (entry + (count.max() / 16 + 8) * 2.0 ** -24) * reach
        assert ((dq[part].double() - want).abs() <= off + step * (want.abs() + off)).all()
    total, reach = (by * a).sum().item() / n, (by * a.abs()).sum().item() / n
    hits = torch.zeros(n, dtype=torch.float64, device="cuda").index_add_(0, t.long().clamp(min=0), by * a)
    for at in range(0, n, 1 << 19):
        part = slice(at, at + (1 << 19))
        want, all_of = (total - hits[part])[:, None], (reach + hits[part])[:, None]
        off = (entry + (6 * nq / 16 + 8) * 2.0 ** -24) * all_of
        assert ((dv[part].double() - want).abs() <= off + step * (want.abs() + off)).all()


@pytest.mark.parametrize("dtype,nq,n,d", [("f32", 3, 1200001, 1000), ("bf16", 5, 600001, 1001), ("bf16", 300, 400001, 331), ("f32", 64, 140001, 200), ("f32", 900, 70001, 65)])
def test_many_rows_within_what_their_sums_can_lose(torch, ops, dtype, nq, n, d):
    """Random rows.  A logit is one float32 sum of d products (six of parts each in float32), rounded once for every eight of them at most: dz.  A lane adds no more
    than 512 exponentials before the joins (no fewer than 512 workgroups share the rows of these sizes): 512 half steps.  dq is summed over ranges of the rows, no
fewer than fill 256 workgroups with tiles of 128 x 128, in the same steps of eight products."""
    kind = torch.float32 if dtype == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(nq + d)
    v = torch.randn((n, d), generator=g, device="cuda", dtype=kind) / 32
    q = torch.randn((nq, d), generator=g, device="cuda", dtype=kind) / 2
    t = torch.randint(0, n, (nq,), generator=g, device="cuda").int()
    t[-1] = n - 1
    w = torch.rand(nq, generator=g, device="cuda") + 0.5
    scale, parts, step = 2.0, (6 if dtype == "f32" else 1), half_step(dtype)
    loss, lse = ops.softmax_loss(q, v, t, scale)
    dq, dv = ops.softmax_loss_grad(q, v, t, scale, lse, w, loss=loss)
    q64, rows = q.double(), 1 << 17
    total, reach, high = torch.zeros(nq, dtype=torch.float64, device="cuda"), 0.0, 0.0
    for at in range(0, n, rows):
        x = v[at:at + rows].double()
        z = scale * (q64 @ x.t())
        total += torch.exp(z).sum(1)
        reach, high = max(reach, scale * (q64.abs() @ x.abs().t()).max().item()), max(high, z.abs().max().item())
    want = total.log()
    dz = (parts * d / 8 + 2) * 2.0 ** -23 * reach + 4 * 2.0 ** -24 * (2 * high + want.abs().max().item())
    de = dz + 2.0 ** -22 + 512 * 2.0 ** -24
    assert (lse - want).abs().max().item() <= de
    hit = scale * (q64 * v[t.long()].double()).sum(1)
    assert ((loss - (want - hit)).abs() <= de + dz).all()
    by = (w * scale).double()[:, None]
    sum_q, off_q = torch.zeros((nq, d), dtype=torch.float64, device="cuda"), torch.zeros((nq, d), dtype=torch.float64, device="cuda")
    r = step if dtype == "bf16" else 2.0 ** -23
    chain = n / max(1, 256 // (-(-nq // 128) * -(-d // 128)))
    for at in range(0, n, rows):
        x = v[at:at + rows].double()
        p = torch.exp(scale * (q64 @ x.t()) - want[:, None]) * by
        hits = torch.zeros_like(p)
        here = (t >= at) & (t < at + rows)
        hits[here, (t[here] - at).long()] = by[here, 0]
        gr, dg = p - hits, (2 * de + dz) * p
        dg = dg + r * (gr.abs() + dg)
        sum_q += gr @ x
        off_q += dg @ x.abs() + (parts * chain / 8 + 260) * 2.0 ** -23 * (gr.abs() @ x.abs())   # (and the join of the ranges)
        one = gr.t() @ q64
        off = dg.t() @ q64.abs() + (parts * nq / 8 + 4) * 2.0 ** -23 * (gr.abs().t() @ q64.abs())
        assert ((dv[at:at + rows].double() - one).abs() <= off + step * (one.abs() + off)).all()
    assert ((dq.double() - sum_q).abs() <= off_q + step * (sum_q.abs() + off_q)).all()
