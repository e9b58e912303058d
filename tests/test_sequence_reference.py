"""The plain 64-bit gradients of the sequence operators against central differences of the plain forward forms, and the
host-side parts of the operators (frequencies, checks that need no GPU)."""
import ctypes

import numpy as np
import pytest

import primitiv_amd as pa
from primitiv_amd import _lib
from sequence_reference import Attention, Rotary, places

STEP = 1e-5
# Central differences of smooth functions of order 1: the third derivative leaves STEP^2 (1e-10) and the subtraction
# 2^-53 * |sum| / STEP (about 1e-9 for sums up to 100), each times a few hundred terms of order 1.
TOL = 1e-6


def _differences(loss, x):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        old = x[i]
        x[i] = old + STEP
        up = loss()
        x[i] = old - STEP
        down = loss()
        x[i] = old
        g[i] = (up - down) / (2 * STEP)
    return g


@pytest.mark.parametrize("causal", (False, True))
@pytest.mark.parametrize("lists", (None, ((3, 0, 1), (4, 2, 1)), ((4, 1, 0), (2, 3, 0))))
def test_attention_gradients(causal, lists):
    rng = np.random.default_rng(1)
    packed = lists is not None and lists[0][0] == 4
    bs, tq, tk = (1, 6, 6) if packed else (3, 3, 4)
    q, k, v = rng.standard_normal((bs, tq, 4, 3)), rng.standard_normal((bs, tk, 2, 3)), rng.standard_normal((bs, tk, 2, 3))
    gy = rng.standard_normal(q.shape)
    seqs = places(bs, tq, tk, *(lists or (None, None)), packed)
    run = lambda g=None: Attention(q, k, v, seqs, causal, 0.7, "f32", g)  # noqa: E731
    got = run(gy)
    for x, g in ((q, got.gq), (k, got.gk), (v, got.gv)):
        assert np.abs(_differences(lambda: (run().y * gy).sum(), x) - g).max() < TOL


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("norm", (False, True))
def test_rotary_gradients(interleaved, norm):
    rng = np.random.default_rng(2)
    x, gy, w = rng.standard_normal((2, 3, 2, 7)), rng.standard_normal((2, 3, 2, 7)), rng.standard_normal(7)
    freqs = np.float32([1.0, 0.3])
    args = (places(2, 3, 3, (3, 1), (5, 1)), freqs, "f32", interleaved, 2, 1.5)
    run = lambda g=None: Rotary(x, *args, w if norm else None, 1e-2, g)  # noqa: E731
    got = run(gy)
    assert np.abs(_differences(lambda: (run().y * gy).sum(), x) - got.gx).max() < TOL
    if norm:
        assert np.abs(_differences(lambda: (run().y * gy).sum(), w) - got.gw).max() < TOL


def test_rotary_frequencies():
    f, a = pa.rotary_frequencies(4)
    assert a == 1.0 and f.dtype == np.float32
    assert np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-7)
    assert np.allclose(pa.rotary_frequencies(4, method="linear", factor=4.0)[0], f / 4, rtol=1e-6)
    g, _ = pa.rotary_frequencies(4, method="base", factor=8.0)
    assert g[0] == 1.0 and np.isclose(g[-1], f[-1] / 8, rtol=1e-6) and np.all(g <= f)
    g, a = pa.rotary_frequencies(64, method="parts", factor=4.0, original_length=4096)
    f, _ = pa.rotary_frequencies(64)
    turns = 4096 * f.astype(np.float64) / (2 * np.pi)
    assert np.allclose(g[turns > 32], f[turns > 32]) and np.allclose(g[turns < 1], f[turns < 1] / 4)
    assert np.all(np.diff(g) < 0) and np.isclose(a, 0.1 * np.log(4) + 1)
    for bad in (dict(pairs=0), dict(pairs=4, base=1.0), dict(pairs=4, factor=0.5), dict(pairs=4, method="other"),
                dict(pairs=4, method="parts", factor=2.0)):
        with pytest.raises(pa.Error):
            pa.rotary_frequencies(**bad)


def test_calls_without_a_context_are_refused():
    l = _lib.lib()
    seqs = ctypes.c_void_p()
    one = (ctypes.c_uint32 * 1)(1)
    assert l.phip_sequences_create(None, one, None, 1, 0, ctypes.byref(seqs)) == _lib.PHIP_ERR_INVALID_ARGUMENT
    assert l.phip_sequences_destroy(None) == _lib.PHIP_OK
    for kind in ("f32", "f16", "bf16"):
        for name in ("rotary_fw", "rotary_bw", "norm_rotary_fw", "norm_rotary_bw", "attention_fw", "attention_bw"):
            fn = getattr(l, "phip_%s_%s" % (name, kind))
            values = [None if t in (_lib._vp, ctypes.POINTER(ctypes.c_float)) else 1 for t in fn.argtypes]
            assert fn(*values) == _lib.PHIP_ERR_INVALID_ARGUMENT and b"null context" in l.phip_last_error()
