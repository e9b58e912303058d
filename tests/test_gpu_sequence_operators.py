"""Rotary positions, head norms with rotation, and attention through the device front, against plain 64-bit forms with
bounds counted from the roundings (sequence_reference.py)."""
import ctypes

import numpy as np
import pytest

import primitiv_amd as pa
from primitiv_amd import _lib
from sequence_reference import Attention, HALF, Rotary, TINY, places
from util import round_to_storage

pytestmark = pytest.mark.gpu

S = pa.Shape
KINDS = ("f32", "f16", "bf16")


@pytest.fixture(scope="module")
def devices():
    devs = {"f32": pa.HIP(0), "f16": pa.HIP16(0, storage="f16"), "bf16": pa.HIP16(0, storage="bf16")}
    yield devs
    for d in devs.values():
        d.close()


def rounded(x, kind):
    x = np.asarray(x, dtype=np.float32)
    return x if kind == "f32" else round_to_storage(x, kind)


def draw(rng, kind, *shape):
    return rounded(rng.standard_normal(shape), kind)


def tensor(dev, x):
    """[batch, tokens, heads, size] -> [size, heads, tokens] x batch; vectors as they are."""
    shape = S([x.shape[0]]) if x.ndim == 1 else S([x.shape[3], x.shape[2], x.shape[1]], x.shape[0])
    return dev.new_tensor_by_vector(shape, x.reshape(-1))


def check(name, got, want, tol):
    got = np.asarray(got, dtype=np.float64).reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s: %r instead of %r +- %r; worst ratio %.2f" % (
        name, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], np.broadcast_to(tol, want.shape)[bad][0],
        np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)))


# (size, query heads, key heads, tq, tk, batch, q_lens, k_lens, packed, causal)
ATTENTION = {
    "one_token": (64, 8, 8, 1, 1, 1, None, None, False, True),
    "whole": (64, 2, 2, 70, 70, 2, None, None, False, True),
    "not_causal": (64, 2, 1, 33, 65, 2, None, None, False, False),
    "grouped": (128, 8, 2, 130, 130, 1, None, None, False, True),
    "odd_size": (65, 3, 3, 35, 35, 3, None, None, False, True),
    "size_1": (1, 2, 1, 9, 9, 1, None, None, False, True),
    "size_20": (20, 2, 2, 40, 40, 1, None, None, False, True),
    "size_80": (80, 2, 2, 129, 129, 1, None, None, False, True),
    "size_100": (100, 3, 1, 66, 66, 1, None, None, False, False),
    "size_127": (127, 2, 1, 35, 64, 1, None, None, False, True),
    "more_keys": (128, 4, 2, 5, 200, 2, None, None, False, True),
    "fewer_keys_than_queries": (64, 2, 2, 100, 40, 1, None, None, False, True),
    "padded": (64, 4, 2, 96, 96, 5, (96, 1, 0, 64, 33), None, False, True),
    "padded_not_causal": (32, 3, 3, 50, 70, 4, (50, 7, 0, 31), (70, 0, 5, 64), False, False),
    "cache": (128, 8, 2, 1, 300, 6, (1, 1, 1, 1, 0, 1), (300, 1, 63, 64, 9, 65), False, True),
    "cache_new_tokens": (96, 6, 2, 5, 257, 3, (5, 5, 3), (257, 5, 128), False, True),
    "long_cache": (64, 4, 1, 2, 5000, 3, (2, 1, 2), (5000, 1500, 2), False, True),
    "long_cache_odd_size": (33, 3, 3, 1, 2100, 1, None, None, False, False),
    "packed_tokens": (128, 8, 2, 9, 1200, 1, (1, 3, 0, 4), (700, 3, 5, 450), True, True),
    "packed": (64, 4, 2, 200, 200, 1, (70, 1, 0, 64, 65), None, True, True),
    "packed_tail": (128, 4, 4, 160, 170, 1, (33, 1, 64), (40, 0, 97), True, True),
    "packed_many": (32, 2, 1, 300, 300, 1, (1,) * 40 + (0, 3, 130, 2), None, True, False),
    "group_of_3": (64, 9, 3, 45, 45, 2, None, None, False, True),
    "group_of_40": (16, 40, 1, 7, 50, 1, None, None, False, True),
}


def attention_case(rng, kind, name):
    d, hq, hk, tq, tk, bs, q_lens, k_lens, packed, causal = ATTENTION[name]
    q, k, v, gy = (draw(rng, kind, bs, tq, hq, d), draw(rng, kind, bs, tk, hk, d), draw(rng, kind, bs, tk, hk, d),
                   draw(rng, kind, bs, tq, hq, d))
    return q, k, v, gy, places(bs, tq, tk, q_lens, k_lens, packed), causal, q_lens, k_lens, packed


@pytest.mark.parametrize("name", sorted(ATTENTION))
@pytest.mark.parametrize("kind", KINDS)
def test_attention(devices, kind, name):
    dev = devices[kind]
    rng = np.random.default_rng(len(name) * 7 + KINDS.index(kind))
    q, k, v, gy, seqs, causal, q_lens, k_lens, packed = attention_case(rng, kind, name)
    scale = 1.0 / float(np.sqrt(q.shape[3]))
    want = Attention(q, k, v, seqs, causal, scale, kind, gy)
    # tokens outside the sequences hold what a cache or a padded batch may hold
    used_q, used_k = np.zeros(q.shape[:2], bool), np.zeros(k.shape[:2], bool)
    for b, aq, n, ak, m in seqs:
        used_q[b, aq:aq + n] = used_k[b, ak:ak + m] = True
    q[~used_q], k[~used_k], v[~used_k], gy[~used_q] = np.nan, np.nan, np.inf, np.nan
    tq, tk, tv, tg = (tensor(dev, x) for x in (q, k, v, gy))
    lists = None if q_lens is None else dev.new_sequences(q_lens, k_lens, packed)
    y, stats = dev.attention_fw(tq, tk, tv, causal, None, lists, stats=True)
    check("y", y.to_vector(), want.y, want.tol_y)
    got = stats.to_vector().reshape(want.stats.shape)
    assert np.array_equal(np.isneginf(got), np.isneginf(want.stats))
    some = ~np.isneginf(want.stats)
    check("stats", got[some], want.stats[some], want.tol_stats[some])
    assert np.array_equal(dev.attention_fw(tq, tk, tv, causal, scale, lists).to_vector(), y.to_vector())
    # gradients, written over noted zeros and added into what is there
    start = {n: draw(rng, kind, *x.shape) for n, x in (("gq", q), ("gk", k), ("gv", v))}
    for add in (False, True):
        g = {n: tensor(dev, x) if add else dev.new_tensor_by_constant(S([x.shape[3], x.shape[2], x.shape[1]], x.shape[0]), 0)
             for n, x in start.items()}
        dev.attention_bw(tq, tk, tv, y, tg, stats, causal, scale, lists, g["gq"], g["gk"], g["gv"])
        for n in ("gq", "gk", "gv"):
            r, t = getattr(want, n), getattr(want, "tol_" + n)
            if add:
                r, t = r + start[n], t + HALF[kind] * (np.abs(r + start[n]) + t) + TINY[kind]
            check(n + (" added" if add else ""), g[n].to_vector(), r, t)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_one_tensor(devices, kind):
    """The same tensor as queries, keys and values, with its one gradient."""
    dev = devices[kind]
    rng = np.random.default_rng(3)
    x, gy = draw(rng, kind, 2, 75, 2, 64), draw(rng, kind, 2, 75, 2, 64)
    want = Attention(x, x, x, places(2, 75, 75), True, 0.125, kind, gy)
    t = tensor(dev, x)
    y, stats = dev.attention_fw(t, t, t, True, 0.125, None, stats=True)
    g = dev.new_tensor_by_constant(t.shape(), 0)
    dev.attention_bw(t, t, t, y, tensor(dev, gy), stats, True, 0.125, None, g, g, g)
    total = want.gq + want.gk + want.gv
    # each of the three is added and rounded in turn
    tol = want.tol_gq + want.tol_gk + want.tol_gv + HALF[kind] * (np.abs(want.gq) + np.abs(want.gq + want.gk) + np.abs(total)) * 1.05
    check("g", g.to_vector(), total, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_bits_repeat(devices, kind):
    dev = devices[kind]
    rng = np.random.default_rng(4)
    q, k, v, gy = (draw(rng, kind, 1, 300, 4, 64), draw(rng, kind, 1, 300, 2, 64), draw(rng, kind, 1, 300, 2, 64),
                   draw(rng, kind, 1, 300, 4, 64))
    t = [tensor(dev, x) for x in (q, k, v, gy)]
    seen = []
    for _ in range(3):
        y, stats = dev.attention_fw(*t[:3], stats=True)
        g = [dev.new_tensor_by_constant(x.shape(), 0) for x in t[:3]]
        dev.attention_bw(*t[:3], y, t[3], stats, True, 0.125, None, *g)
        seen.append([x.to_vector() for x in (y, *g)])
    for other in seen[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(seen[0], other))


ROTARY = {
    # size, query heads, key heads, tokens, batch, pairs, interleaved, first, q_lens, k_lens, packed
    "one_token": (64, 8, 8, 1, 1, 32, False, 5, None, None, False),
    "whole": (128, 4, 2, 33, 2, 64, False, 0, None, None, False),
    "interleaved": (128, 4, 2, 33, 2, 64, True, 0, None, None, False),
    "part": (64, 3, 1, 17, 1, 8, False, 100000, None, None, False),
    "part_interleaved": (64, 3, 1, 17, 1, 16, True, 1 << 30, None, None, False),
    "odd_size": (65, 10, 10, 35, 3, 16, False, 0, None, None, False),
    "odd_interleaved": (65, 2, 1, 35, 3, 32, True, -7, None, None, False),
    "size_2": (2, 1, 1, 9, 1, 1, False, 0, None, None, False),
    "size_100": (100, 3, 3, 40, 1, 50, False, 0, None, None, False),
    "size_100_quarter": (100, 3, 3, 40, 1, 25, True, 0, None, None, False),
    "no_pairs": (64, 2, 2, 5, 1, 0, False, 0, None, None, False),
    "no_keys": (64, 5, 0, 19, 1, 32, False, 0, None, None, False),
    "padded": (80, 4, 2, 40, 4, 40, False, 0, (40, 0, 1, 17), (1000000, 3, 1, 16), False),
    "packed": (128, 4, 2, 100, 1, 64, True, 3, (0, 33, 0, 1, 50, 0), (7, 40, 0, 12345, 50, 1), True),
    "many_tokens": (32, 3, 1, 5000, 2, 16, False, 0, None, None, False),
}


@pytest.mark.parametrize("norm", (False, True))
@pytest.mark.parametrize("name", sorted(ROTARY))
@pytest.mark.parametrize("kind", KINDS)
def test_rotary(devices, kind, name, norm):
    dev = devices[kind]
    d, hq, hk, t, bs, pairs, inter, first, q_lens, k_lens, packed = ROTARY[name]
    rng = np.random.default_rng(len(name) * 11 + KINDS.index(kind))
    freqs, amplitude = pa.rotary_frequencies(pairs) if pairs else (np.zeros(0, np.float32), 1.0)
    if name == "whole":
        amplitude = 1.25
    seqs = places(bs, t, t, q_lens, k_lens, packed) if q_lens else places(bs, t, t)
    lists = None if q_lens is None else dev.new_sequences(q_lens, k_lens, packed)
    eps = 1e-3
    ops, want = {}, {}
    for n, h in (("q", hq), ("k", hk)):
        if h == 0:
            ops[n] = want[n] = None
            continue
        x, gy, w = draw(rng, kind, bs, t, h, d), draw(rng, kind, bs, t, h, d), rounded(1 + 0.2 * rng.standard_normal(d), kind)
        ops[n] = [tensor(dev, a) for a in (x, gy, w)]
        want[n] = Rotary(x, seqs, freqs, kind, inter, first, amplitude, w if norm else None, eps if norm else 0, gy)
    part = lambda i: [None if ops[n] is None else ops[n][i] for n in ("q", "k")]  # noqa: E731
    if norm:
        got = dev.norm_rotary_fw(*part(0), *part(2), freqs, eps, inter, first, amplitude, lists)
    else:
        got = dev.rotary_fw(*part(0), freqs, inter, first, amplitude, lists)
    for n, y in zip(("q", "k"), got):
        if want[n] is not None:
            check("y" + n, y.to_vector(), want[n].y, want[n].tol_y)
    for add in (False, True):
        g, start = {}, {}
        for n in ("q", "k"):
            if want[n] is not None:
                for key, like in (("x", ops[n][0]), ("w", ops[n][2])):
                    start[key + n] = draw(rng, kind, like.shape().size()) * (1.0 if add else 0.0)
                    g[key + n] = dev.new_tensor_by_vector(like.shape(), start[key + n]) if add else dev.new_tensor_by_constant(like.shape(), 0)
        if norm:
            dev.norm_rotary_bw(*part(0), *part(2), *part(1), freqs, eps, inter, first, amplitude, lists, g["xq"], g.get("xk"),
                               g["wq"], g.get("wk"))
        else:
            dev.rotary_bw(*part(1), freqs, inter, first, amplitude, lists, g["xq"], g.get("xk"))
        for key in g:
            if key[0] == "w" and not norm:
                continue
            r, tol = getattr(want[key[1]], "g" + key[0]), getattr(want[key[1]], "tol_g" + key[0])
            if add:
                r = r + start[key].reshape(r.shape)
                tol = tol + HALF[kind] * (np.abs(r) + tol) + TINY[kind]
            check("g" + key, g[key].to_vector(), r, tol)


@pytest.mark.parametrize("norm", (False, True))
@pytest.mark.parametrize("kind", KINDS)
def test_rotary_of_one_tensor(devices, kind, norm):
    """One tensor as queries and keys, one weight for both: each gradient passed twice."""
    dev = devices[kind]
    rng = np.random.default_rng(5)
    x, gq, gk = (draw(rng, kind, 2, 21, 3, 64) for _ in range(3))
    w = rounded(1 + 0.2 * rng.standard_normal(64), kind)
    freqs, _ = pa.rotary_frequencies(32)
    a, b = (Rotary(x, places(2, 21, 21), freqs, kind, w=w if norm else None, eps=1e-6, gy=gy) for gy in (gq, gk))
    t, tw, tq, tk = (tensor(dev, z) for z in (x, w, gq, gk))
    g, gw = dev.new_tensor_by_constant(t.shape(), 0), dev.new_tensor_by_constant(tw.shape(), 0)
    if norm:
        dev.norm_rotary_bw(t, t, tw, tw, tq, tk, freqs, 1e-6, False, 0, 1.0, None, g, g, gw, gw)
        check("gw", gw.to_vector(), a.gw + b.gw, a.tol_gw + b.tol_gw + 1.05 * HALF[kind] * (np.abs(a.gw) + np.abs(a.gw + b.gw)))
    else:
        dev.rotary_bw(tq, tk, freqs, False, 0, 1.0, None, g, g)
    check("gx", g.to_vector(), a.gx + b.gx, a.tol_gx + b.tol_gx + 1.05 * HALF[kind] * (np.abs(a.gx) + np.abs(a.gx + b.gx)))
