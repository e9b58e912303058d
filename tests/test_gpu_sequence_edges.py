"""Sequence operators where their inputs, sizes or addresses are unusual: against the plain 64-bit forms, with bounds counted
from the roundings (sequence_reference.py)."""
import ctypes

import numpy as np
import pytest

import primitiv_amd as pa
from primitiv_amd import _lib
from sequence_reference import Attention, HALF, Rotary, TINY, places
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


# Shapes of which every call fills the chip several times over with 128-row tiles, forward, over queries and over keys:
# (size, query heads, key heads, tq, tk, batch, q_lens, k_lens, packed, causal)
LARGE = {
    "whole": (64, 16, 8, 150, 150, 20, None, None, False, True),
    "not_causal": (128, 8, 8, 70, 200, 35, None, None, False, False),
    "grouped": (128, 12, 4, 300, 300, 25, None, None, False, True),
    "size_1": (1, 8, 4, 140, 140, 40, None, None, False, True),
    "size_5": (5, 8, 8, 130, 70, 40, None, None, False, False),
    "size_20": (20, 9, 3, 200, 200, 50, None, None, False, True),
    "size_33": (33, 8, 8, 99, 99, 35, None, None, False, True),
    "size_65": (65, 10, 10, 135, 135, 20, None, None, False, True),
    "size_66": (66, 8, 4, 150, 170, 40, None, None, False, True),
    "size_95": (95, 6, 6, 140, 140, 25, None, None, False, False),
    "size_127": (127, 8, 8, 90, 90, 35, None, None, False, True),
    "fewer_keys_than_queries": (64, 8, 8, 200, 80, 35, None, None, False, True),
    "padded": (64, 16, 8, 160, 160, 20, (160, 0, 1, 129, 64) * 4, None, False, True),
    "padded_odd_size": (33, 8, 8, 150, 170, 20, (150, 0, 1, 129, 64) * 4, (3, 170, 5, 64, 129) * 4, False, False),
    "packed": (64, 16, 8, 4200, 4300, 1, (70, 1, 0, 350, 128, 700) * 3, (70, 2, 9, 350, 0, 700) * 3, True, True),
    "packed_odd_size": (65, 12, 12, 3000, 3000, 1, (70, 1, 0, 350, 128, 400) * 3, None, True, True),
    "group_of_40": (16, 160, 4, 40, 140, 35, None, None, False, True),
    "many_keys": (64, 8, 8, 70, 1100, 35, None, None, False, True),
    "many_keys_odd_size": (65, 4, 4, 70, 1030, 70, None, None, False, True),
}


def attention_against_reference(dev, kind, shape, seed, kernels):
    """Forward and gradients of one shape; `kernels`: what each of the three must have gone to."""
    d, hq, hk, tq, tk, bs, q_lens, k_lens, packed, causal = shape
    rng = np.random.default_rng(seed)
    q, k, v, gy = (draw(rng, kind, bs, t, h, d) for t, h in ((tq, hq), (tk, hk), (tk, hk), (tq, hq)))
    seqs = places(bs, tq, tk, q_lens, k_lens, packed)
    scale = 1.0 / float(np.sqrt(d))
    want = Attention(q, k, v, seqs, causal, scale, kind, gy)
    used_q, used_k = np.zeros(q.shape[:2], bool), np.zeros(k.shape[:2], bool)
    for b, aq, n, ak, m in seqs:
        used_q[b, aq:aq + n] = used_k[b, ak:ak + m] = True
    q[~used_q], k[~used_k], v[~used_k], gy[~used_q] = np.nan, np.nan, np.inf, np.nan
    tq_, tk_, tv_, tg_ = (tensor(dev, x) for x in (q, k, v, gy))
    lists = None if q_lens is None else dev.new_sequences(q_lens, k_lens, packed)
    start = {n: draw(rng, kind, *x.shape) for n, x in (("gq", q), ("gk", k), ("gv", v))}
    g = {n: tensor(dev, x) for n, x in start.items()}
    dev.gemm_trace(True)
    y, stats = dev.attention_fw(tq_, tk_, tv_, causal, scale, lists, stats=True)
    dev.attention_bw(tq_, tk_, tv_, y, tg_, stats, causal, scale, lists, g["gq"], g["gk"], g["gv"])
    went = dev.gemm_trace(False)
    assert [w.replace("_fix", "") for w in went] == list(kernels), went
    # the rounding of y in delta is taken out for 16-bit storage and up to 64 keys
    assert went[1].endswith("_fix") == (kind != "f32" and max(k_lens or q_lens or (tk,)) <= 64)
    check("y", y.to_vector(), want.y, want.tol_y)
    got = stats.to_vector().reshape(want.stats.shape)
    assert np.array_equal(np.isneginf(got), np.isneginf(want.stats))
    some = ~np.isneginf(want.stats)
    check("stats", got[some], want.stats[some], want.tol_stats[some])
    for n in ("gq", "gk", "gv"):
        r, t = getattr(want, n) + start[n], getattr(want, "tol_" + n)
        check(n, g[n].to_vector(), r, t + HALF[kind] * (np.abs(r) + t) + TINY[kind])
    zeroed = {n: dev.new_tensor_by_constant(t.shape(), 0) for n, t in (("gq", tq_), ("gk", tk_), ("gv", tv_))}
    dev.attention_bw(tq_, tk_, tv_, y, tg_, stats, causal, scale, lists, zeroed["gq"], zeroed["gk"], zeroed["gv"])
    for n in ("gq", "gk", "gv"):
        check(n + " over zeros", zeroed[n].to_vector(), getattr(want, n), getattr(want, "tol_" + n))
    return went


@pytest.mark.parametrize("name", sorted(LARGE))
@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_tiles_of_128_rows(devices, kind, name):  # noqa: F811
    """The kernels whose workgroups share tiles, which prompts and training go to."""
    attention_against_reference(devices[kind], kind, LARGE[name], 30 + len(name),
                                ("attention_rows", "attention_queries", "attention_keys"))


# Up to 64 keys: 16-bit storage takes the rounding of the stored result out of the queries' gradients
FEW_KEYS = {
    "size_64": (64, 16, 8, 150, 64, 40, None, None, False, False),
    "size_65": (65, 8, 8, 130, 50, 40, None, None, False, True),
    "size_128": (128, 8, 8, 70, 64, 40, (70, 0, 1, 64) * 10, (64, 33, 1, 64) * 10, False, True),
}


@pytest.mark.parametrize("name", sorted(FEW_KEYS))
@pytest.mark.parametrize("kind", KINDS[1:])
def test_attention_with_tiles_of_128_rows_and_few_keys(devices, kind, name):  # noqa: F811
    went = attention_against_reference(devices[kind], kind, FEW_KEYS[name], 50 + len(name),
                                       ("attention_rows", "attention_queries", "attention_keys"))
    assert went[1] == "attention_queries_fix"


# Short sequences, so many that every SIMD has one: in fp32 a wavefront each
SHORT = {
    "whole": (64, 16, 16, 35, 35, 33, None, None, False, True),
    "odd_size": (65, 10, 10, 35, 35, 64, None, None, False, True),
    "size_1": (1, 16, 16, 50, 50, 33, None, None, False, False),
    "size_33": (33, 16, 16, 64, 64, 33, None, None, False, True),
    "grouped": (128, 32, 16, 20, 31, 40, None, None, False, True),
    "padded": (96, 16, 16, 60, 64, 36, (60, 0, 1, 33) * 9, (60, 9, 3, 64) * 9, False, True),
    "packed": (80, 40, 40, 400, 430, 1, (33, 1, 0, 60, 17) * 3, (35, 1, 9, 64, 0) * 3, True, True),
}


@pytest.mark.parametrize("name", sorted(SHORT))
def test_attention_with_a_wavefront_per_tile(devices, name):  # noqa: F811
    attention_against_reference(devices["f32"], "f32", SHORT[name], 60 + len(name),
                                ("attention_few1", "attention_few1_queries", "attention_few1_keys"))


@pytest.mark.parametrize("size", (64, 65))
@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_tiles_of_128_rows_before_a_value_that_is_no_number(devices, kind, size):  # noqa: F811
    dev = devices[kind]
    rng = np.random.default_rng(7)
    bs, n, h = 20, 150, 8
    q, k, v = (draw(rng, kind, bs, n, h, size) for _ in range(3))
    want = Attention(q, k, v, places(bs, n, n), True, 0.125, kind)
    first = 100   # rows from here on see it; it lies in the middle of a tile of keys
    v[:, first, :, 5] = np.nan
    v[:, first + 3, :, 7] = np.inf
    k[:, n - 1] = np.nan
    dev.gemm_trace(True)
    y = dev.attention_fw(tensor(dev, q), tensor(dev, k), tensor(dev, v), True, 0.125).to_vector().reshape(want.y.shape)
    assert dev.gemm_trace(False) == ["attention_rows"]
    check("y", y[:, :first], want.y[:, :first], want.tol_y[:, :first])
    assert np.isnan(y[:, first:, :, 5]).all() and not np.isfinite(y[:, first + 3:, :, 7]).any()
    others = [i for i in range(size) if i not in (5, 7)]
    check("other columns", y[:, first:-1][..., others], want.y[:, first:-1][..., others], want.tol_y[:, first:-1][..., others])
    assert np.isnan(y[:, -1]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_one_tensor_with_tiles_of_128_rows(devices, kind):  # noqa: F811
    """The same tensor as queries, keys and values, with its one gradient; the same bits on every run."""
    dev = devices[kind]
    rng = np.random.default_rng(8)
    x, gy = draw(rng, kind, 35, 135, 8, 64), draw(rng, kind, 35, 135, 8, 64)
    want = Attention(x, x, x, places(35, 135, 135), True, 0.125, kind, gy)
    t, tg = tensor(dev, x), tensor(dev, gy)
    seen = []
    for _ in range(3):
        dev.gemm_trace(True)
        y, stats = dev.attention_fw(t, t, t, True, 0.125, None, stats=True)
        g = dev.new_tensor_by_constant(t.shape(), 0)
        dev.attention_bw(t, t, t, y, tg, stats, True, 0.125, None, g, g, g)
        went = [w.replace("_fix", "") for w in dev.gemm_trace(False)]
        assert went == ["attention_rows", "attention_queries", "attention_keys"]
        seen.append((y.to_vector(), g.to_vector()))
    for other in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(seen[0], other))
    total = want.gq + want.gk + want.gv
    tol = want.tol_gq + want.tol_gk + want.tol_gv + HALF[kind] * (np.abs(want.gq) + np.abs(want.gq + want.gk) + np.abs(total)) * 1.05
    check("g", seen[0][1], total, tol)


# fp16 holds 2^-24 .. 65504; probabilities of thousands of keys, and these times gradients, need not lie in it.
# (queries, keys, heads, batch): few tiles, and tiles of 128 rows
SCALED = {"few": (24, 6000, 2, 1), "large": (16, 4096, 8, 17)}


@pytest.mark.parametrize("name", sorted(SCALED))
@pytest.mark.parametrize("size_gy", (1e-2, 1e-3, 2e-4))
@pytest.mark.parametrize("wide", ("q", "k"))
def test_fp16_gradients_of_many_keys_lose_no_range(devices, wide, size_gy, name):  # noqa: F811
    """gq and gk from a dS far below fp16's normal range, where gy and the gradients are in it.

    dS = P (dP - delta) is rounded once for the matrix instructions, by at most h = 2^-11 of itself, with signs that are
    independent of each other: what they add to an element of gq has a root mean square of at most
    h scale sqrt(sum_j (dS k)^2), and likewise for gk.  The stored y (off by at most h of itself) adds an error to delta
    whose root mean square is h sqrt(sum gy^2 y^2), and that, times P, one to dS; the result is rounded once (h of itself, or
    half of fp16's smallest step, 2^-25).  fp32 roundings are 2^-12 of these.  All of these are upper bounds of the single
    errors, so that the measured root mean square has to stay below their sum (in fact about 1 / sqrt(3) of it)."""
    dev = devices["f16"]
    n, m, heads, bs = SCALED[name]
    d, scale, h = 64, 0.125, 2.0 ** -11
    rng = np.random.default_rng(21)
    q, k, v, gy = (draw(rng, "f16", bs, t, heads, d) for t in (n, m, m, n))
    # scores of order 1, and the operand that the wanted gradient is a sum of is large: the gradient is in fp16's range
    q, k = (rounded(x * (32.0 if wide == w else 1 / 32.0), "f16") for x, w in ((q, "q"), (k, "k")))
    gy = rounded(gy * size_gy, "f16")
    t = [tensor(dev, x) for x in (q, k, v, gy)]
    dev.gemm_trace(True)
    y, stats = dev.attention_fw(*t[:3], False, scale, None, stats=True)
    g = [dev.new_tensor_by_constant(x.shape(), 0) for x in t[:3]]
    dev.attention_bw(*t[:3], y, t[3], stats, False, scale, None, *g)
    assert ("attention_queries" in dev.gemm_trace(False)) == (name == "large")
    got = [x.to_vector().astype(np.float64).reshape(z.shape) for x, z in zip(g, (q, k, v))]
    q, k, v, gy = (x.astype(np.float64) for x in (q, k, v, gy))
    error, bound = [], []
    for b in range(bs):
        for a in range(heads):
            Q, K, V, G = (x[b, :, a] for x in (q, k, v, gy))
            P = np.exp(scale * Q @ K.T)
            P /= P.sum(1, keepdims=True)
            Y, dP = P @ V, G @ V.T
            dS = P * (dP - (G * Y).sum(1)[:, None])
            at_delta = P * (h * np.sqrt((G * G * Y * Y).sum(1)))[:, None]
            if wide == "k":   # gq
                want, parts = scale * dS @ K, scale * np.sqrt((dS * dS) @ (K * K))
                delta = scale * np.abs(at_delta @ K)
                error.append(got[0][b, :, a] - want)
            else:             # gk
                want, parts = scale * dS.T @ Q, scale * np.sqrt((dS * dS).T @ (Q * Q))
                delta = scale * np.sqrt((at_delta * at_delta).T @ (Q * Q))
                error.append(got[1][b, :, a] - want)
            own = np.maximum(h * np.abs(want), 2.0 ** -25)
            assert np.sqrt((want * want).mean()) > 2.0 ** -19, "the gradient itself is out of range"
            bound.append(np.sqrt((h * parts) ** 2 + delta ** 2 + own ** 2))
    error, bound = (np.sqrt((np.stack(x) ** 2).mean()) for x in (error, bound))
    assert error <= bound, "%.3g, %.2f times the bound" % (error, error / bound)


@pytest.mark.parametrize("name", ("few", "large"))
def test_fp16_gradients_beyond_the_largest_number_on_the_way(devices, name):  # noqa: F811
    """dS above 65504 where the gradients are below it."""
    dev = devices["f16"]
    rng = np.random.default_rng(22)
    n, heads, bs = (40, 2, 1) if name == "few" else (70, 8, 35)
    q, k, v, gy = (draw(rng, "f16", bs, n, heads, 64) for _ in range(4))
    q, k, v, gy = (rounded(x * f, "f16") for x, f in ((q, 1 / 16), (k, 1 / 16), (v, 8), (gy, 6000)))
    seqs = places(bs, n, n)
    want = Attention(q, k, v, seqs, True, 0.125, "f16", gy)
    t = [tensor(dev, x) for x in (q, k, v, gy)]
    y, stats = dev.attention_fw(*t[:3], True, 0.125, None, stats=True)
    g = [dev.new_tensor_by_constant(x.shape(), 0) for x in t[:3]]
    dev.attention_bw(*t[:3], y, t[3], stats, True, 0.125, None, *g)
    s = q[0, :, 0].astype(np.float64) @ k[0, :, 0].T * 0.125
    p = np.where(np.tril(np.ones((n, n), bool)), np.exp(s), 0)
    p /= p.sum(1, keepdims=True)
    dp = gy[0, :, 0].astype(np.float64) @ v[0, :, 0].T
    dS = np.abs(p * (dp - (p * dp).sum(1, keepdims=True))).max()
    assert dS > 65504 > max(np.abs(want.gq).max(), np.abs(want.gk).max(), np.abs(want.gv).max())
    # of a dS scaled so that the largest of a block is 2^12 or more, the smallest step is 2^-36 of that largest one
    step = 2.0 ** -37 * 4 * dS * 0.125 * n * max(np.abs(q).max(), np.abs(k).max())
    for x, r in zip(g, ("gq", "gk", "gv")):
        check(r, x.to_vector(), getattr(want, r), getattr(want, "tol_" + r) + (step if r != "gv" else 0))


@pytest.mark.parametrize("name,shape", (("few", (4, 2, 4096, 1)), ("split", (1, 1, 8192, 1)), ("large", (130, 8, 1500, 18))))
def test_fp16_many_small_probabilities_beside_a_large_one(devices, name, shape):  # noqa: F811
    """One key takes nearly all of the weight, with a value of zero: the result is what thousands of keys with weights of
    2^-26 each add up to.  Rounded once each (h of itself), and the result once."""
    dev = devices["f16"]
    n, heads, m, bs = shape
    rng = np.random.default_rng(23)
    q, k, v = np.zeros((bs, n, heads, 64)), np.zeros((bs, m, heads, 64)), 32 + 4 * rng.standard_normal((bs, m, heads, 64))
    q[..., 0], k[:, 5, :, 0], v[:, 5] = 1.0, 18.0, 0.0
    k[..., 1] = rng.standard_normal(k.shape[:-1])
    q[..., 1] = 0.25
    q, k, v = (rounded(x, "f16") for x in (q, k, v))
    want = Attention(q, k, v, places(bs, n, m), False, 1.0, "f16")
    dev.gemm_trace(True)
    y, stats = dev.attention_fw(*(tensor(dev, x) for x in (q, k, v)), False, 1.0, None, stats=True)
    went = dev.gemm_trace(False)
    assert went == [{"few": "attention_few_split", "split": "attention_few_split", "large": "attention_rows"}[name]]
    # two halves of a step; scores of 18 are off by 70 x 2^-24 x 18 at most
    check("y", y.to_vector(), want.y, np.abs(want.y) * (2 * 2.0 ** -11 + 2.0 ** -13) + 2.0 ** -25)
    check("stats", stats.to_vector(), want.stats.reshape(-1), want.tol_stats.reshape(-1))


def test_one_gradient_for_operands_of_different_shapes_is_refused(devices):  # noqa: F811
    """The gradient of queries is that of keys (or values) only where they have the same heads and tokens."""
    dev = devices["f32"]
    ones = lambda n: dev.new_tensor_by_constant(S([n]), 1)  # noqa: E731
    for hq, hk, tq, tk in ((4, 2, 6, 6), (2, 2, 6, 7), (2, 2, 7, 6), (4, 4, 6, 6)):
        q, k, y, g, other = ones(64 * hq * tq), ones(64 * hk * tk), ones(64 * hq * tq), ones(64 * 4 * 8), ones(64 * 4 * 8)
        stats = ones(hq * tq)
        for gq, gk, gv in ((g, g, other), (g, other, g), (g, g, g), (other, g, g)):
            before = [x.to_vector() for x in (g, other)]
            rc = _lib.lib().phip_attention_bw_f32(
                dev.ctx(), q.handle(), k.handle(), k.handle(), y.handle(), stats.handle(), y.handle(), gq.handle(), gk.handle(),
                gv.handle(), 64, hq, hk, tq, tk, 1, None, 1, 0.125)
            if (hq, tq) == (hk, tk) or gq is other:
                assert rc == _lib.PHIP_OK
            else:
                assert rc == _lib.PHIP_ERR_INVALID_ARGUMENT and b"overlap" in _lib.lib().phip_last_error()
                assert all(np.array_equal(a, x.to_vector()) for a, x in zip(before, (g, other)))


def test_stats_in_another_tensor_or_at_an_odd_address_are_refused(devices):  # noqa: F811
    dev = devices["f32"]
    q, k, v, y = (dev.new_tensor_by_constant(S([64, h, 6], 2), 1) for h in (4, 2, 2, 4))
    own = dev.new_tensor_by_constant(S([4 * 6 * 2 + 4]), 5)
    call = lambda stats: _lib.lib().phip_attention_fw_f32(  # noqa: E731
        dev.ctx(), q.handle(), k.handle(), v.handle(), y.handle(), stats, 64, 4, 2, 6, 6, 2, None, 1, 0.125)
    for x in (q, k, v, y):
        for stats in (x.handle(), x.handle() + 4 * (x.shape().size() - 1), x.handle() - 4 * 47):
            assert call(stats) == _lib.PHIP_ERR_INVALID_ARGUMENT and b"share" in _lib.lib().phip_last_error()
    for o in (1, 2, 3):
        assert call(own.handle() + o) == _lib.PHIP_ERR_INVALID_ARGUMENT and b"multiple" in _lib.lib().phip_last_error()
    assert all((x.to_vector() == c).all() for x, c in ((q, 1), (k, 1), (v, 1), (y, 1), (own, 5)))
    assert call(own.handle() + 4) == _lib.PHIP_OK
    assert (own.to_vector()[[0, -3, -2, -1]] == 5).all() and (own.to_vector()[1:-3] != 5).all()


@pytest.mark.parametrize("kind", KINDS)
def test_rotary_at_an_odd_address_is_refused(devices, kind):  # noqa: F811
    dev = devices[kind]
    f = (ctypes.c_float * 32)()
    size = 64 * 2 * 5
    block = dev.new_tensor_by_constant(S([8 * size]), 1)
    rest = (64, 2, 2, 5, 1, None, 0, f, 32, 0, 1.0)
    for norm in (False, True):
        for back in (False, True):
            n = (10 if norm else 4) if back else (6 if norm else 4)
            name = "phip_%srotary_%s_%s" % ("norm_" if norm else "", "bw" if back else "fw", kind)
            good = [block.handle() + dev._ITEMSIZE * (size * i if i < 6 else 6 * size + 64 * i) for i in range(n)]
            for odd in range(n):
                args = [p + (1 if i == odd else 0) for i, p in enumerate(good)]
                rc = getattr(_lib.lib(), name)(dev.ctx(), *args, *rest, *((1e-6,) if norm else ()))
                assert rc == _lib.PHIP_ERR_INVALID_ARGUMENT and b"multiple" in _lib.lib().phip_last_error(), (name, odd)
    assert (block.to_vector() == 1).all()


def test_rotary_of_more_tokens_than_a_launch_has_threads_for():
    """2^27 tokens and a few: 256 threads for every eight of them would be more than 2^32."""
    dev = pa.HIP16(0, storage="f16")
    tokens = 2 ** 27 + 13
    x = dev.new_tensor_by_constant(S([2, 1, tokens]), 1)
    freqs = np.float32([2.0 ** -10])
    y, _ = dev.rotary_fw(x, None, freqs)
    g = dev.new_tensor_by_constant(x.shape(), 0)
    dev.rotary_bw(x, None, freqs, False, 0, 1.0, None, g, None)
    for at in (0, 1000, 2 ** 26 + 5, 2 ** 27 - 3, tokens - 8):
        p = (np.arange(at, at + 8) * float(freqs[0]))
        for t, sign in ((y, 1), (g, -1)):
            got = np.empty(16, np.float16)
            _lib.call("phip_memcpy_d2h", dev.ctx(), got.ctypes.data, t.handle() + 4 * at, 32)
            want = np.stack([np.cos(p) - sign * np.sin(p), np.cos(p) + sign * np.sin(p)], 1)
            # fp32 cosines and sines (8 x 2^-24 of a sum of at most 2) and one rounding
            check("at %d" % at, got, want, 2.0 ** -11 * np.abs(want) + 2.0 ** -20 + TINY["f16"])
    del x, y, g
    dev.close()


def test_attention_of_more_sequences_than_a_launch_has_threads_for_is_refused():
    dev = pa.HIP16(0, storage="f16")
    n = 2 ** 24
    x = dev.new_tensor_by_constant(S([1, 1, 1], n), 1)
    with pytest.raises(pa.Error, match="too many rows"):
        dev.attention_fw(x, x, x)
    y, stats = dev.attention_fw(*(dev.new_tensor_by_constant(S([1, 1, 1], n - 1), 1) for _ in range(3)), stats=True)
    assert (y.to_vector() == 1).all()
    big = dev.new_tensor_by_constant(S([n]), 1)
    g = dev.new_tensor_by_constant(x.shape(), 0)
    rc = _lib.lib().phip_attention_bw_f16(dev.ctx(), x.handle(), x.handle(), x.handle(), x.handle(), _pool(dev, 4 * n), big.handle(),
                                          g.mutable_handle(), g.mutable_handle(), g.mutable_handle(), 1, 1, 1, 1, 1, n, None, 1, 1.0)
    assert rc == _lib.PHIP_ERR_INVALID_ARGUMENT and b"too many rows" in _lib.lib().phip_last_error()
    assert (g.to_vector() == 0).all()   # a gradient that was to be zero is
    del x, y, stats, big, g
    dev.close()


def _pool(dev, size):
    ptr = ctypes.c_void_p()
    _lib.call("phip_pool_alloc", dev.ctx(), size, ctypes.byref(ptr), None)
    return ptr.value


def test_attention_of_very_many_fp32_sequences():
    """In fp32 short sequences take a wavefront each: four times as many as workgroups of four wavefronts could be."""
    dev = pa.HIP(0)
    n = 2 ** 24 + 5
    q, k, v = (dev.new_tensor_by_constant(S([1, 1, 1], n), x) for x in (1, 2, 3))
    y, stats = dev.attention_fw(q, k, v, scale=0.5, stats=True)
    g = [dev.new_tensor_by_constant(q.shape(), 0) for _ in range(3)]
    dev.attention_bw(q, k, v, y, v, stats, True, 0.5, None, *g)
    for t, want in ((y, 3), (stats, 1), (g[0], 0), (g[1], 0), (g[2], 3)):
        assert (t.to_vector() == want).all()
    del q, k, v, y, stats, g
    dev.close()


# Lists of which one sequence is much longer than the others: workgroups only for ranges of keys that exist
LISTED = {
    "packed_one_long": (128, 8, 1, 140, 28200, 1, (1,) * 128, (64,) * 100 + (20000,) + (64,) * 27, True, True),
    "packed_some_empty": (64, 8, 2, 40, 9000, 1, (1, 0, 3, 1, 0, 2, 1) * 4, (10, 4000, 3, 0, 0, 400, 1000) + (10, 300, 3, 0, 0, 400, 100) * 3, True, True),
    "packed_not_causal": (33, 2, 2, 30, 8000, 1, (1, 2) * 10, (7000, 1) + (1, 7) * 9, True, False),
    "padded_one_long": (64, 8, 2, 1, 7000, 20, (1,) * 20, (7, 7000, 0, 300, 64) + (100,) * 15, False, True),
    "padded_five_tokens": (128, 16, 2, 5, 5000, 12, (5, 0, 3) * 4, (5000, 9, 1) + (5, 600, 2) * 3, False, True),
    "padded_odd_size": (65, 6, 2, 2, 4000, 9, (2, 1, 2) * 3, (30, 4000, 700) + (2, 1, 0) * 2, False, False),
}


@pytest.mark.parametrize("name", sorted(LISTED))
@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_one_long_sequence_among_short_ones(devices, kind, name):  # noqa: F811
    dev = devices[kind]
    d, hq, hk, tq, tk, bs, q_lens, k_lens, packed, causal = LISTED[name]
    rng = np.random.default_rng(80 + len(name))
    q, k, v = (draw(rng, kind, bs, t, h, d) for t, h in ((tq, hq), (tk, hk), (tk, hk)))
    seqs = places(bs, tq, tk, q_lens, k_lens, packed)
    scale = 1.0 / float(np.sqrt(d))
    want = Attention(q, k, v, seqs, causal, scale, kind)
    used_q, used_k = np.zeros(q.shape[:2], bool), np.zeros(k.shape[:2], bool)
    for b, aq, n, ak, m in seqs:
        used_q[b, aq:aq + n] = used_k[b, ak:ak + m] = True
    q[~used_q], k[~used_k], v[~used_k] = np.nan, np.nan, np.inf
    t = [tensor(dev, x) for x in (q, k, v)]
    lists = dev.new_sequences(q_lens, k_lens, packed)
    seen = []
    for _ in range(3):   # the tickets are left as they were found
        dev.gemm_trace(True)
        y, stats = dev.attention_fw(*t, causal, scale, lists, stats=True)
        assert dev.gemm_trace(False) == ["attention_few_listed"]
        seen.append(y.to_vector())
        check("y", seen[-1], want.y, want.tol_y)
        got = stats.to_vector().reshape(want.stats.shape)
        assert np.array_equal(np.isneginf(got), np.isneginf(want.stats))
        some = ~np.isneginf(want.stats)
        check("stats", got[some], want.stats[some], want.tol_stats[some])
    assert np.array_equal(seen[0], seen[1]) and np.array_equal(seen[0], seen[2])


def test_memory_of_one_long_sequence_among_short_ones():
    """Partial results for the ranges that exist: some 10 MB, not for the longest's ranges of every sequence."""
    dev = pa.HIP16(0, storage="bf16")
    hip = ctypes.CDLL("libamdhip64.so")
    free, total = ctypes.c_size_t(), ctypes.c_size_t()

    def left():
        _lib.call("phip_sync", dev.ctx())
        assert hip.hipMemGetInfo(ctypes.byref(free), ctypes.byref(total)) == 0
        return free.value
    lens = [131072] + [64] * 127
    q, k = dev.new_tensor_by_constant(S([128, 8, len(lens)]), 1), dev.new_tensor_by_constant(S([128, 1, sum(lens)]), 1)
    lists, y = dev.new_sequences([1] * len(lens), lens, True), dev.attention_fw(q, k, k)
    before = left()
    y = dev.attention_fw(q, k, k, True, None, lists)
    assert before - left() < 64 << 20
    assert (y.to_vector() == 1).all()
    del q, k, y, lists
    dev.close()


@pytest.mark.parametrize("lens,kernel", (
    ((4096,) * 16, "attention_few_split"), ((4096,) * 17, "attention_few"), ((4096,) * 31, "attention_few"),
    ((4096,) * 40, "attention_few"), ((8192,) + (512,) * 30, "attention_few_listed"), ((8192,) + (512,) * 31, "attention_few_listed"),
    ((8192,) + (512,) * 63, "attention_few_listed"), ((8192,) * 4 + (1000,) * 60, "attention_few_split")))
def test_keys_are_cut_by_the_lengths_not_by_the_number_of_streams(lens, kernel):
    dev = pa.HIP16(0, storage="bf16")
    n = len(lens)
    q, k = dev.new_tensor_by_constant(S([128, 32, 1], n), 1), dev.new_tensor_by_constant(S([128, 8, max(lens)], n), 1)
    lists = dev.new_sequences((1,) * n, lens)
    dev.gemm_trace(True)
    y, stats = dev.attention_fw(q, k, k, True, 0.01, lists, stats=True)
    assert dev.gemm_trace(False) == [kernel]
    assert (y.to_vector() == 1).all()
    # scores of 1.28: fp32 sums of up to 8192 equal terms
    check("stats", stats.to_vector().reshape(n, 32), np.repeat(1.28 + np.log(np.float64(lens))[:, None], 32, 1), 1e-4)
    del q, k, y, stats, lists
    dev.close()


@pytest.mark.parametrize("tokens,keys,batch,one", ((8, 8, 64, True), (8, 8, 63, False), (32, 256, 64, True), (32, 257, 64, False),
                                                   (35, 35, 64, True), (35, 35, 63, False), (65, 65, 128, False)))
def test_which_fp32_sequences_take_a_wavefront_each(devices, tokens, keys, batch, one):  # noqa: F811
    """From 512 tiles of 32 rows on, or from 1024 on where they are two to a sequence or walk far."""
    dev = devices["f32"]
    q, k = (dev.new_tensor_by_constant(S([16, 8, t], batch), 1) for t in (tokens, keys))
    dev.gemm_trace(True)
    y = dev.attention_fw(q, k, k)
    assert (dev.gemm_trace(False) == ["attention_few1"]) == one
    # the weights and the weighted ones are added up apart (half a step a term), then divided
    assert np.abs(y.to_vector() - 1).max() <= (2 * keys + 2) * 2.0 ** -24


@pytest.mark.parametrize("kind", KINDS[1:])
@pytest.mark.parametrize("shape", ((1, 300, 64, 8, 2, 3), (4, 2000, 128, 16, 4, 1), (1, 700, 65, 3, 3, 2)))
def test_single_tokens_in_16_bits_lose_nothing_but_the_results_rounding(devices, kind, shape):  # noqa: F811
    """Where a sequence's rows are one tile, the probabilities keep twice the storage type's bits."""
    dev, h = devices[kind], HALF[kind]
    tq, tk, d, hq, hk, bs = shape
    rng = np.random.default_rng(90 + tk)
    q, k, v = (draw(rng, kind, bs, t, n, d) for t, n in ((tq, hq), (tk, hk), (tk, hk)))
    args = (places(bs, tq, tk), True, 0.125, kind)
    want, size = Attention(q, k, v, *args), Attention(q, k, np.abs(v), *args).y   # size: the sum of |P v|
    y = dev.attention_fw(*(tensor(dev, x) for x in (q, k, v)), True, 0.125)
    # the bound allows one rounding (h) of each probability: what is left of it is the rounding of the second part, h h
    check("y", y.to_vector(), want.y, want.tol_y - 1.05 * (h - h * h) * size)


# Groups larger than a tile of rows, up to the largest: (heads, batch, kernels of bf16)
@pytest.mark.parametrize("kind,heads,batch,kernels", (
    ("f32", 1024, 1, ("attention_few", "attention_few_queries", "attention_few_keys")),
    ("f16", 300, 1, ("attention_few", "attention_few_queries", "attention_few_keys")),
    ("bf16", 1024, 6, ("attention_rows", "attention_queries", "attention_few_keys"))))
def test_attention_of_large_groups(devices, kind, heads, batch, kernels):  # noqa: F811
    attention_against_reference(devices[kind], kind, (16, heads, 1, 3, 40, batch, None, None, False, True), 100, kernels)


def test_a_larger_group_is_refused(devices):  # noqa: F811
    dev = devices["f32"]
    q, k = (dev.new_tensor_by_constant(S([16, h, 2]), 1) for h in (1025, 1))
    with pytest.raises(pa.Error, match="1024 query heads"):
        dev.attention_fw(q, k, k)


@pytest.mark.parametrize("shape", ((128, 33, 1, 7, 400, 1, None, None, False, True), (64, 10, 2, 200, 1500, 1, None, None, False, True),
                                   (64, 8, 8, 70, 300, 35, None, None, False, True)))
@pytest.mark.parametrize("size", (1.0, 300.0))
def test_fp16_gradients_with_scores_of_hundreds(devices, shape, size):  # noqa: F811
    """Probabilities from 2^-140 to 1 in one row: the first block of keys may have hardly any weight, the next nearly all."""
    dev = devices["f16"]
    d, hq, hk, tq, tk, bs = shape[:6]
    rng = np.random.default_rng(0)
    q, k, v, gy = (rounded(rng.standard_normal((bs, t, h, d)) * f, "f16") for t, h, f in (
        (tq, hq, 6), (tk, hk, 6), (tk, hk, 1), (tq, hq, size)))
    want = Attention(q, k, v, places(bs, tq, tk), True, 1.0, "f16", gy)
    t = [tensor(dev, x) for x in (q, k, v, gy)]
    y, stats = dev.attention_fw(*t[:3], True, 1.0, None, stats=True)
    g = [dev.new_tensor_by_constant(x.shape(), 0) for x in t[:3]]
    dev.attention_bw(*t[:3], y, t[3], stats, True, 1.0, None, *g)
    # dS is rounded to half of a step of 2^-24 where its largest is 2^13 or more: 2^-38 of the largest, at most 2 d |gy| |v|
    step = 2.0 ** -38 * 2 * d * np.abs(gy).max() * np.abs(v).max() * max(np.abs(q).max(), np.abs(k).max()) * max(tk, tq * hq // hk)
    for x, n in zip((y, *g), ("y", "gq", "gk", "gv")):
        r = getattr(want, n)
        assert np.abs(r).max() < 65504
        check(n, x.to_vector(), r, getattr(want, "tol_" + n) + (step if n in ("gq", "gk") else 0))


def test_packed_tokens_at_far_positions(devices):  # noqa: F811
    """The lengths of keys are positions to the rotary operators: their sum has no limit.  Attention needs the keys."""
    dev = devices["f32"]
    rng = np.random.default_rng(24)
    q_lens, k_lens = (2, 3, 1), (2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30)
    x, freqs = draw(rng, "f32", 1, 6, 2, 64), pa.rotary_frequencies(32)[0]
    lists = dev.new_sequences(q_lens, k_lens, True)
    y, _ = dev.rotary_fw(tensor(dev, x), None, freqs, seqs=lists)
    want = Rotary(x, places(1, 6, 6, q_lens, k_lens, True), freqs, "f32")
    # the angle's product, in 64 bits: half a step each of it and of the turns, at 2^31 radians 2^-21 in all
    check("y", y.to_vector(), want.y, want.tol_y + 2.0 ** -21 * np.abs(x).max() * 2)
    t = tensor(dev, x)
    with pytest.raises(pa.Error, match="packed sequences"):
        dev.attention_fw(t, t, t, seqs=lists)
