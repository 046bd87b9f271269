"""Refusals of the training and 8-bit scoring operators that need no GPU, and their plain implementations against each other."""
import ctypes

import numpy as np
import pytest

import ops_support as ref


def test_params_struct_layout_matches_header(pkg):
    p = pkg.binding.JvSoftmaxParams
    assert ctypes.sizeof(p) == 88
    assert p.scale.offset == 24 and p.queries.offset == 32 and p.vectors.offset == 48 and p.targets.offset == 64 and p.workspace_bytes.offset == 80


def test_bad_arguments_are_refused_before_any_device_is_touched(pkg):
    b = pkg.binding
    A = 4096   # an aligned address that nothing reads
    good = dict(device=0, vec=A, dtype=0, stride=64, n=10, d=64, codes=A, scales=A)

    def encode(**kw):
        g = {**good, **kw}
        return lambda: b.encode_blocks_device(g["device"], g["vec"], g["dtype"], g["stride"], g["n"], g["d"], g["codes"], g["scales"])

    def decode(**kw):
        g = {**good, **kw}
        return lambda: b.decode_blocks_device(g["device"], g["codes"], g["scales"], g["n"], g["d"], g["dtype"], g["vec"], g["stride"])

    def score(**kw):
        g = {**good, "stride": 10, "nq": 3, **kw}
        return lambda: b.score_blocks_device(g["device"], g["codes"], g["scales"], g["nq"], g["codes"], g["scales"], g["n"], g["d"], g["dtype"], g["vec"], g["stride"])

    wrong = []
    for f in (encode, decode):
        wrong += [f(dtype=2), f(dtype=-1), f(n=-1), f(d=0), f(d=-3), f(vec=0), f(vec=A + 1), f(vec=A + 2), f(stride=63), f(stride=(1 << 31) + 1), f(codes=0), f(scales=0),
                  f(codes=A + 8)]
    wrong += [score(nq=-1), score(n=-1), score(d=0), score(stride=9), score(vec=0), score(codes=A + 1), score(scales=0), score(dtype=7)]
    for k, call in enumerate(wrong):
        with pytest.raises(b.JvError) as e:
            call()
        assert e.value.code == b.JV_EINVAL, k
    for call in (encode(d=b.OPS_MAX_D + 1, stride=1 << 20), encode(n=2 ** 31 - 1), score(nq=2 ** 31 - 1), score(n=2 ** 31 - 100, stride=1 << 31)):
        with pytest.raises(b.JvError) as e:
            call()
        assert e.value.code == b.JV_EUNSUPPORTED


def test_bad_softmax_arguments_are_refused_before_any_device_is_touched(pkg):
    b = pkg.binding
    A, B = 1 << 20, 1 << 40

    def params(**kw):
        p = b.softmax_params(0, kw.pop("dtype", 1), kw.pop("nq", 5), kw.pop("n", 100), kw.pop("d", 64), kw.pop("scale", 1.0), A, 64, A, 64, A)
        p.workspace, p.workspace_bytes = A, B
        for k, x in kw.items():
            setattr(p, k, x)
        return p

    def both(**kw):
        return [lambda: b.softmax_loss_device(params(**kw), A, A), lambda: b.softmax_grad_device(params(**kw), A, A, A, 64, A, 64)]

    wrong = [c for kw in (dict(struct_size=80), dict(dtype=3), dict(nq=-1), dict(n=-1), dict(d=0), dict(scale=float("inf")), dict(scale=float("nan")), dict(queries=None),
                          dict(vectors=None), dict(queries=A + 1), dict(query_stride=63), dict(vector_stride=0), dict(workspace=None), dict(workspace=A + 16),
                          dict(workspace_bytes=255)) for c in both(**kw)]
    wrong += [lambda: b.softmax_loss_device(params(), 0, A), lambda: b.softmax_loss_device(params(), A, 0), lambda: b.softmax_grad_device(params(), 0, A, A, 64, A, 64),
              lambda: b.softmax_grad_device(params(), A, A, 0, 64, 0, 64), lambda: b.softmax_grad_device(params(), A, A, A, 63, 0, 0),
              lambda: b.softmax_grad_device(params(), A, A, 0, 0, A + 1, 64), lambda: b.softmax_workspace(params(), 0), lambda: b.softmax_workspace(params(), 8)]
    for k, call in enumerate(wrong):
        with pytest.raises(b.JvError) as e:
            call()
        assert e.value.code == b.JV_EINVAL, k
    for kw in (dict(d=b.OPS_MAX_D + 1), dict(n=2 ** 31 - 1), dict(nq=b.SOFTMAX_MAX_QUERIES + 1)):
        with pytest.raises(b.JvError) as e:
            b.softmax_workspace(params(**kw), 7)
        assert e.value.code == b.JV_EUNSUPPORTED


def test_workspace_follows_the_shape_alone_and_one_for_both_calls_is_enough(pkg):
    b = pkg.binding
    for dtype in (0, 1):
        for nq, n, d in ((0, 0, 1), (1, 1, 1), (16, 10000, 128), (1000, 70001, 381), (4096, 131072, 1024), (4096, 10 ** 8, 64)):
            p = b.softmax_params(0, dtype, nq, n, d, 1.0)
            each = [b.softmax_workspace(p, w) for w in (1, 2, 4, 6)]
            assert b.softmax_workspace(p, 7) == max(each) and min(each) >= 256 and all(x % 256 == 0 for x in each)
            # far from the logits: at most the laid-out operands of one piece, whatever n is
            if n >= 10 ** 8:
                assert max(each) < nq * n * 4 // 100


def test_the_plain_implementations(pkg):
    """The float64 gradient against differences, the encoder against its decoder: every code comes back."""
    rng = np.random.default_rng(3)
    q, v, t, w = rng.standard_normal((4, 6)), rng.standard_normal((9, 6)), np.array([0, 3, -1, 3]), rng.random(4)
    out = ref.softmax(q, v, t, 1.5, w, "f32")
    total = lambda q, v: float((w * ref.softmax(q, v, t, 1.5, w, "f32")["loss"][0]).sum())  # noqa: E731
    for x, g, f in ((q, out["dq"][0], lambda y: total(y, v)), (v, out["dv"][0], lambda y: total(q, y))):
        for i in np.ndindex(x.shape):
            y = x.copy()
            y[i] += 1e-5
            up = f(y)
            y[i] -= 2e-5
            assert abs((up - f(y)) / 2e-5 - g[i]) < 1e-8
    codes = np.tile(np.arange(127, dtype=np.uint8), (3, 1))
    codes = np.concatenate([codes, np.full((3, 1), 126, np.uint8)], 1)
    scales = np.array([[0], [127], [240]], np.uint8)
    back = ref.encode(ref.decode(codes, scales, 128))
    assert np.array_equal(back[0], codes) and np.array_equal(back[1], scales)
