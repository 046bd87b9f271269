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
