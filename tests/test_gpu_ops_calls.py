"""What calls of the training operators ask of memory, autograd and the caller."""
import importlib

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module("opensearch_jvector_amd.ops")


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("nq,mib", [(1, 16), (16, 128)])
def test_rows_that_are_not_laid_out_get_no_room(torch, ops, nq, mib):
    """The gradient of aligned bf16 rows allocates what it uses: a few copies of g (nq x n x 2 bytes), not the rows (768 MiB here)."""
    n, d = 524288, 768
    g = torch.Generator(device="cuda").manual_seed(1)
    v = torch.randn((n, d), generator=g, device="cuda", dtype=torch.bfloat16)
    q, t = v[:nq].clone(), torch.arange(nq, device="cuda", dtype=torch.int32)
    loss, lse = ops.softmax_loss(q, v, t, 0.05)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    dq, _ = ops.softmax_loss_grad(q, v, t, 0.05, lse, vectors_grad=False, loss=loss)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < mib << 20
    # the same rows, one component further on, are laid out: the same gradient but for where the sums are cut
    wide = torch.zeros(n * d + 1, dtype=torch.bfloat16, device="cuda")
    moved = wide[1:].view(n, d)
    moved.copy_(v)
    again, _ = ops.softmax_loss_grad(q, moved, t, 0.05, lse, vectors_grad=False, loss=loss)
    # (the same g; float32 sums in chains of some 400 products, 2^-15 of the reach, which is about the largest component; one rounding each)
    assert ((again.double() - dq.double()).abs() <= 2 * 2.0 ** -8 * dq.double().abs() + 2.0 ** -12 * dq.double().abs().max()).all()


def test_a_loss_that_autograd_would_not_see_is_refused(torch, ops):
    q, v = torch.randn(4, 32, device="cuda", requires_grad=True), torch.randn(9, 32, device="cuda", requires_grad=True)
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    want = ops.softmax_loss(q.detach(), v.detach(), t, 1.0)
    for args in ((q, v), (q, v.detach()), (q.detach(), v), (q * 2, v.detach())):
        with pytest.raises(ValueError, match="autograd"):
            ops.softmax_loss(*args, t, 1.0)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(ops.softmax_loss(q, v, t, 1.0), want))
    with torch.inference_mode():
        assert torch.equal(ops.softmax_loss(q, v, t, 1.0)[0], want[0])
    # the gradient is what a caller hands on: no graph is expected of it
    loss, lse = want
    dq, dv = ops.softmax_loss_grad(q, v, t, 1.0, lse, loss=loss)
    q.backward(dq)
    assert torch.equal(q.grad, dq) and not dq.requires_grad and not dv.requires_grad


def case(torch, dtype, nq=50, n=1500, d=100):
    g = torch.Generator(device="cuda").manual_seed(nq + n + d)
    v = torch.randn((n, d), generator=g, device="cuda") / d ** 0.5
    t = torch.randint(0, n, (nq,), generator=g, device="cuda").int()
    q = v[t.long()] + torch.randn((nq, d), generator=g, device="cuda") / d ** 0.5 / 4
    t[::6] = -1
    return q.to(dtype), v.to(dtype), t, torch.rand(nq, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_entry_without_losses_is_the_one_with_none(torch, ops, pkg, dtype):
    import ctypes
    b = pkg.binding
    q, v, t, w = case(torch, torch.float32 if dtype == "f32" else torch.bfloat16)
    loss, lse = ops.softmax_loss(q, v, t, 12.0)
    want = ops.softmax_loss_grad(q, v, t, 12.0, lse, w)
    p = b.softmax_params(0, b.DTYPE_F32 if dtype == "f32" else b.DTYPE_BF16, *q.shape[:1], *v.shape, 12.0, q.data_ptr(), 100, v.data_ptr(), 100, t.data_ptr())
    p.workspace_bytes = b.softmax_workspace(p, 6)
    ws = torch.empty(p.workspace_bytes, dtype=torch.uint8, device="cuda")
    p.workspace = ws.data_ptr()
    dq, dv = torch.full_like(q, float("nan")), torch.full_like(v, float("nan"))
    torch.cuda.synchronize()
    assert b.load_library().jv_softmax_grad_device(ctypes.byref(p), lse.data_ptr(), w.data_ptr(), dq.data_ptr(), 100, dv.data_ptr(), 100, None) == b.JV_OK
    assert torch.equal(dq, want[0]) and torch.equal(dv, want[1])
    with_loss = ops.softmax_loss_grad(q, v, t, 12.0, lse, w, loss=loss)
    assert not torch.equal(with_loss[1], want[1])   # (the losses are looked at)


def step(torch, ops, q, v, t, w):
    loss, lse = ops.softmax_loss(q, v, t, 12.0)
    return (loss, lse, *ops.softmax_loss_grad(q, v, t, 12.0, lse, w, loss=loss))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n,d", [(50, 1500, 100), (40, 300, 700), (90, 36000, 130), (300, 30011, 200)])
def test_a_captured_step_with_its_losses_replays(torch, ops, dtype, nq, n, d):
    q, v, t, w = case(torch, torch.float32 if dtype == "f32" else torch.bfloat16, nq, n, d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(torch, ops, q, v, t, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(torch, ops, q, v, t, w)
    for k in range(4):
        q.mul_(1.0 + 0.125 * k)
        t.copy_(t.roll(1))
        for x in out:
            x.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step(torch, ops, q, v, t, w))), k


def test_two_steps_with_their_losses_at_once(torch, ops):
    cases = [case(torch, kind, nq, 5000, 96) for kind, nq in ((torch.float32, 40), (torch.bfloat16, 200), (torch.float32, 300))]
    want = [step(torch, ops, *c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(3):
        for s, c, runs in zip(streams, cases, got):
            with torch.cuda.stream(s):
                runs.append(step(torch, ops, *c))
    torch.cuda.synchronize()
    for x, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(x, r))
