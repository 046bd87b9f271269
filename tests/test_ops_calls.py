"""What the entry points of the training and 8-bit scoring operators take and refuse, without a GPU."""
import pytest


def test_a_scale_whose_base_2_form_passes_float32_is_refused(pkg):
    """The kernels multiply by scale log2(e): above 2.36e38 that is infinite, and every logit would be NaN, those of 0 too."""
    b = pkg.binding
    A = 1 << 20
    for scale in (3.4e38, -3.4e38, 2.4e38):
        p = b.softmax_params(0, b.DTYPE_F32, 5, 100, 64, scale, A, 64, A, 64, A)
        p.workspace, p.workspace_bytes = A, 1 << 40
        for call in (lambda: b.softmax_loss_device(p, A, A), lambda: b.softmax_grad_device(p, A, A, A, 64, A, 64), lambda: b.softmax_workspace(p, 7)):
            with pytest.raises(b.JvError) as e:
                call()
            assert e.value.code == b.JV_EINVAL
    for scale in (2.35e38, -2.35e38, 0.0, 1e-45):
        assert b.softmax_workspace(b.softmax_params(0, b.DTYPE_F32, 5, 100, 64, scale), 7) > 0


def test_a_workspace_for_vectors_as_they_lie(pkg):
    """Aligned bf16 rows are not laid out: no room for that.  Any others, and a shape alone, need what they needed."""
    b = pkg.binding

    def need(nq, n, d, what, vectors=0, stride=0, dtype=b.DTYPE_BF16):
        return b.softmax_workspace(b.softmax_params(0, dtype, nq, n, d, 1.0, 0, 0, vectors, stride), what)

    here = b.SOFTMAX_AS_THEY_LIE
    for nq, most in ((1, 16 << 20), (16, 128 << 20), (256, 1 << 30)):
        for what in (1, 2, 4, 7):
            shape = need(nq, 1000000, 768, what)
            lain = need(nq, 1000000, 768, what | here, 4096, 768)
            assert lain < most and lain <= shape
            for vectors, stride in ((4098, 768), (4096, 769)):   # laid out
                assert need(nq, 1000000, 768, what | here, vectors, stride) == shape
            assert need(nq, 1000000, 768, what, 4096, 768) == shape
            for d, dtype in ((767, b.DTYPE_BF16), (768, b.DTYPE_F32), (3, b.DTYPE_F32)):   # never, or always, laid out
                assert need(nq, 1000, d, what | here, 4096, 768, dtype) == need(nq, 1000, d, what, 0, 0, dtype)
    for what in (here, 0, 16, 17, 16 | here):
        with pytest.raises(b.JvError) as e:
            need(1, 10, 8, what)
        assert e.value.code == b.JV_EINVAL
