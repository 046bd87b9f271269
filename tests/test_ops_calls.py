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


def test_the_gradient_without_losses_refuses_what_the_one_with_them_refuses(pkg):
    """jv_softmax_grad_device itself (the binding calls jv_softmax_grad_device_ex)."""
    import ctypes
    b = pkg.binding
    lib, A = b.load_library(), 1 << 20

    def call(name, params, lse=A, dq=A, dq_stride=64, dv=A, dv_stride=64):
        between = (None,) if name.endswith("_ex") else ()
        return getattr(lib, name)(ctypes.byref(params), lse, *between, None, dq, dq_stride, dv, dv_stride, None)

    def params(**kw):
        p = b.softmax_params(0, kw.pop("dtype", 1), 5, 100, 64, kw.pop("scale", 1.0), A, 64, A, 64, A)
        p.workspace, p.workspace_bytes = A, 1 << 40
        for k, x in kw.items():
            setattr(p, k, x)
        return p
    for name in ("jv_softmax_grad_device", "jv_softmax_grad_device_ex"):
        for kw in (dict(struct_size=80), dict(dtype=3), dict(scale=float("inf")), dict(queries=A + 1), dict(vector_stride=0), dict(workspace=None), dict(workspace_bytes=255)):
            assert call(name, params(**kw)) == b.JV_EINVAL, (name, kw)
        assert call(name, params(), lse=None) == b.JV_EINVAL and call(name, params(), dq=None, dv=None) == b.JV_EINVAL
        assert call(name, params(), dq_stride=63) == b.JV_EINVAL and call(name, params(), dv=A + 1) == b.JV_EINVAL
        assert call(name, params(d=b.OPS_MAX_D + 1)) == b.JV_EUNSUPPORTED


def test_a_float32_workspace_has_room_for_what_is_laid_out_alone(pkg):
    """Rows and queries of fewer than four components are laid out with four (16 bytes), others of few tiles not at all."""
    b = pkg.binding

    def need(nq, n, d, what):
        return b.softmax_workspace(b.softmax_params(0, b.DTYPE_F32, nq, n, d, 1.0), what)
    # 2^15 queries of 2^16 components against 16 rows: taken as they lie; dv's copy of those without a target as zeros is 8 GiB
    nq, d = 1 << 15, 1 << 16
    assert need(nq, 16, d, b.SOFTMAX_LOSS) < 1 << 20
    assert need(nq, 16, d, b.SOFTMAX_QUERY_GRAD) < (nq * d * 4) + (64 << 20)          # one range of dq's partial sums
    assert need(nq, 16, d, b.SOFTMAX_VECTOR_GRAD) < (nq * d * 4) + (64 << 20)
    # rows of three components: no more than 16 bytes each of one piece, and the partial sums
    assert need(64, 6000001, 3, b.SOFTMAX_LOSS) < 6000001 * 16
    assert need(1, 1000, 3, b.SOFTMAX_LOSS) < 1000 * 16 + 8192
