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
