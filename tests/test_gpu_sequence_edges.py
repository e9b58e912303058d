"""Sequence operators where their inputs, sizes or addresses are unusual: against the plain 64-bit forms, with bounds counted
from the roundings (sequence_reference.py)."""
import numpy as np
import pytest

import primitiv_amd as pa
from sequence_reference import HALF, Rotary, TINY, places
from test_gpu_sequence_operators import KINDS, check, devices, draw, rounded, tensor  # noqa: F401

pytestmark = pytest.mark.gpu

S = pa.Shape


# (q_lens, packed): padded samples of 9 tokens, one of them empty; packed sequences with tokens behind the last one
@pytest.mark.parametrize("lens,packed", (((9, 0, 4), False), ((5, 0, 13), True)))
@pytest.mark.parametrize("add", (False, True))
@pytest.mark.parametrize("kind", KINDS)
def test_norm_without_eps_beside_tokens_of_no_sequence(devices, kind, add, lens, packed):  # noqa: F811
    """eps = 0: a token of no sequence, whose root mean square may be 0, adds nothing to any gradient."""
    dev = devices[kind]
    rng = np.random.default_rng(20)
    bs, t, d, freqs = (1, 27, 64, pa.rotary_frequencies(32)[0]) if packed else (3, 9, 64, pa.rotary_frequencies(32)[0])
    seqs = places(bs, t, t, lens, None, packed)
    used = np.zeros((bs, t), bool)
    for b, a, n, _, _ in seqs:
        used[b, a:a + n] = True
    ops, want = {}, {}
    for n, h in (("q", 4), ("k", 2)):
        x, gy, w = draw(rng, kind, bs, t, h, d), draw(rng, kind, bs, t, h, d), rounded(1 + 0.2 * rng.standard_normal(d), kind)
        x[~used] = 0
        ops[n] = [tensor(dev, a) for a in (x, gy, w)]
        with np.errstate(all="ignore"):
            want[n] = Rotary(x, seqs, freqs, kind, w=w, eps=0.0, gy=gy)
    lists = dev.new_sequences(lens, None, packed)
    part = lambda i: [ops[n][i] for n in ("q", "k")]  # noqa: E731
    for n, y in zip(("q", "k"), dev.norm_rotary_fw(*part(0), *part(2), freqs, 0.0, seqs=lists)):
        check("y" + n, y.to_vector(), want[n].y, want[n].tol_y)
    g, start = {}, {}
    for n in ("q", "k"):
        for key, like in (("x", ops[n][0]), ("w", ops[n][2])):
            start[key + n] = draw(rng, kind, like.shape().size()) * (1.0 if add else 0.0)
            g[key + n] = dev.new_tensor_by_vector(like.shape(), start[key + n]) if add else dev.new_tensor_by_constant(like.shape(), 0)
    dev.norm_rotary_bw(*part(0), *part(2), *part(1), freqs, 0.0, False, 0, 1.0, lists, g["xq"], g["xk"], g["wq"], g["wk"])
    for key in g:
        r, tol = getattr(want[key[1]], "g" + key[0]), getattr(want[key[1]], "tol_g" + key[0])
        got = g[key].to_vector()
        if key[0] == "x":
            behind = np.broadcast_to(~used[:, :, None, None], r.shape).reshape(-1)
            assert np.array_equal(got[behind], start[key][behind])
        if add:
            r = r + start[key].reshape(r.shape)
            tol = tol + HALF[kind] * (np.abs(r) + tol) + TINY[kind]
        check("g" + key, got, r, tol)
