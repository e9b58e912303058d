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


@pytest.mark.parametrize("keys,queries,group", ((150, 150, 2), (90, 6, 2), (40, 40, 1)))
@pytest.mark.parametrize("kind", KINDS)
def test_attention_rows_before_a_value_that_is_no_number(devices, kind, keys, queries, group):
    """A key and a value that a row does not see may be anything; the rows that see them are no numbers."""
    dev = devices[kind]
    rng = np.random.default_rng(6)
    q, k, v = draw(rng, kind, 1, queries, 2 * group, 64), draw(rng, kind, 1, keys, 2, 64), draw(rng, kind, 1, keys, 2, 64)
    want = Attention(q, k, v, places(1, queries, keys), True, 0.125, kind)
    first = keys - 4   # seen by the last four queries
    v[0, first, :, 5] = np.nan
    v[0, keys - 2, :, 7] = np.inf
    k[0, keys - 1] = np.nan
    y = dev.attention_fw(tensor(dev, q), tensor(dev, k), tensor(dev, v), True, 0.125).to_vector().reshape(want.y.shape)
    clean = queries - 4
    check("y", y[:, :clean], want.y[:, :clean], want.tol_y[:, :clean])
    assert np.isnan(y[0, clean:, :, 5]).all()
    others = [i for i in range(64) if i not in (5, 7)]
    check("other columns", y[:, clean:-1][..., others], want.y[:, clean:-1][..., others], want.tol_y[:, clean:-1][..., others])
    assert np.isnan(y[0, -1]).all()


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


def test_refusals(devices):
    dev, half = devices["f32"], devices["f16"]
    raw = lambda *dims, batch=1: dev.new_tensor_by_constant(S(list(dims), batch), 1)  # noqa: E731
    q, k = raw(64, 4, 6, batch=2), raw(64, 2, 6, batch=2)
    freqs, _ = pa.rotary_frequencies(32)
    good = dev.new_sequences([6, 3], [6, 6])
    calls = [
        lambda: dev.attention_fw(q, k, raw(64, 2, 7, batch=2)),                      # keys and values differ
        lambda: dev.attention_fw(q, raw(32, 2, 6, batch=2), raw(32, 2, 6, batch=2)),  # sizes differ
        lambda: dev.attention_fw(q, raw(64, 3, 6, batch=2), raw(64, 3, 6, batch=2)),  # 4 heads over 3
        lambda: dev.attention_fw(q, raw(64, 2, 6), raw(64, 2, 6)),                    # batches differ
        lambda: dev.attention_fw(raw(129, 1, 2), raw(129, 1, 2), raw(129, 1, 2)),     # head too large
        lambda: dev.attention_fw(q, k, k, scale=0.0),
        lambda: dev.attention_fw(q, k, k, scale=-1.0),
        lambda: dev.attention_fw(q, k, k, scale=float("nan")),
        lambda: dev.attention_fw(q, k, k, seqs=half.new_sequences([6, 6])),           # another device's list
        lambda: dev.attention_fw(q, k, k, seqs=dev.new_sequences([6, 7])),            # longer than the samples
        lambda: dev.attention_fw(q, k, k, seqs=dev.new_sequences([6, 6], [6, 9])),
        lambda: dev.attention_fw(q, k, k, seqs=dev.new_sequences([6])),               # one list entry, two samples
        lambda: dev.attention_fw(q, k, k, seqs=dev.new_sequences([3, 3], packed=True)),
        lambda: dev.attention_fw(raw(64, 4, 6), raw(64, 2, 6), raw(64, 2, 6), seqs=dev.new_sequences([4, 3], packed=True)),
        lambda: dev.new_sequences([]),
        lambda: dev.new_sequences([1, 2], [1]),
        lambda: dev.new_sequences([-1]),
        lambda: dev.new_sequences([2 ** 31]),
        lambda: dev.rotary_fw(q, raw(64, 2, 5, batch=2), freqs),
        lambda: dev.rotary_fw(q, None, pa.rotary_frequencies(33)[0]),
        lambda: dev.rotary_fw(raw(130, 1, 1), None, freqs),
        lambda: dev.norm_rotary_fw(q, k, raw(64), None, freqs),
        lambda: dev.norm_rotary_fw(q, None, raw(63), None, freqs),
        lambda: dev.norm_rotary_fw(q, None, raw(64), None, freqs, eps=-1.0),
        lambda: dev.attention_fw(half.new_tensor_by_constant(q.shape(), 1), k, k),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(pa.Error):
            call()
            pytest.fail("call %d was not refused" % i)
    y, stats = dev.attention_fw(q, k, k, seqs=good, stats=True)
    g = lambda t: dev.new_tensor_by_constant(t.shape(), 0)  # noqa: E731
    with pytest.raises(pa.Error):   # a gradient where an operand is
        dev.attention_bw(q, k, k, y, y, stats, True, 0.1, good, q, g(k), g(k))
    with pytest.raises(pa.Error):   # stats of another shape
        other = dev.attention_fw(raw(64, 4, 3, batch=2), k, k, stats=True)[1]
        dev.attention_bw(q, k, k, y, y, other, True, 0.1, good, g(q), g(k), g(k))
    # gradients that overlap in part, through the C ABI
    big = raw(64 * 4 * 6 * 4)
    args = (dev.ctx(), q.handle(), k.handle(), k.handle(), y.handle(), stats.handle(), y.handle())
    rc = _lib.lib().phip_attention_bw_f32(*args, big.handle(), big.handle() + 4 * 64, big.handle() + 4 * 64 * 4 * 6 * 3,
                                          64, 4, 2, 6, 6, 2, None, 1, 0.1)
    assert rc == _lib.PHIP_ERR_INVALID_ARGUMENT
    # a gradient that was to be zero is, after a refused call too
    noted = g(k)
    with pytest.raises(pa.Error):
        dev.attention_bw(q, k, k, y, y, stats, True, 0.0, good, g(q), noted, noted)
    assert (noted.to_vector() == 0).all()
    # nothing was enqueued by the refused calls: the device works on
    assert np.isfinite(dev.attention_fw(q, k, k).to_vector()).all()


def test_addresses_that_are_no_multiple_of_16(devices):
    """Tensors inside a larger block: the C ABI takes any address that suits the element."""
    rng = np.random.default_rng(8)
    for kind, offsets in (("f16", (1, 2, 3, 8)), ("bf16", (1, 6)), ("f32", (1, 2, 3))):
        dev = devices[kind]
        q, k, v, gy = (draw(rng, kind, 1, n, h, 64) for n, h in ((50, 4), (70, 2), (70, 2), (50, 4)))
        want = Attention(q, k, v, places(1, 50, 70), True, 0.125, kind, gy)
        for o in offsets:
            def put(x):
                t = dev.new_tensor_by_vector(S([x.size + o]), np.concatenate([np.zeros(o, np.float32), x.reshape(-1)]))
                return t, t.handle() + o * dev._ITEMSIZE
            t = [put(x) for x in (q, k, v, gy, np.zeros_like(q), np.zeros_like(q), np.zeros_like(k), np.zeros_like(v))]
            pq, pk, pv, pg, py, gq, gk, gv = (x[1] for x in t)
            stats = dev._staging(200) if kind != "f32" else dev.new_tensor_by_constant(S([200]), 0)
            ps = stats.ptr if kind != "f32" else stats.handle()
            shape = (64, 4, 2, 50, 70, 1, None, 1, 0.125)
            _lib.call("phip_attention_fw_" + kind, dev.ctx(), pq, pk, pv, py, ps, *shape)
            _lib.call("phip_attention_bw_" + kind, dev.ctx(), pq, pk, pv, py, ps, pg, gq, gk, gv, *shape)
            for i, name in ((4, "y"), (5, "gq"), (6, "gk"), (7, "gv")):
                got = t[i][0].to_vector()
                assert (got[:o] == 0).all()
                check("%s at %d" % (name, o), got[o:], getattr(want, name), getattr(want, "tol_" + name))
            freqs, _ = pa.rotary_frequencies(32)
            r = Rotary(q, places(1, 50, 50), freqs, kind)
            f = freqs.ctypes.data_as(ctypes.POINTER(ctypes.c_float))
            _lib.call("phip_rotary_fw_" + kind, dev.ctx(), pq, None, py, None, 64, 4, 0, 50, 1, None, 0, f, 32, 0, 1.0)
            check("rotary at %d" % o, t[4][0].to_vector()[o:], r.y, r.tol_y)
            # in its operand's place
            _lib.call("phip_rotary_fw_" + kind, dev.ctx(), pq, None, pq, None, 64, 4, 0, 50, 1, None, 0, f, 32, 0, 1.0)
            check("rotary in place", t[0][0].to_vector()[o:], r.y, r.tol_y)


def test_two_devices_at_once(devices):
    """Two contexts on one GPU, calls of both in flight together; lists destroyed while calls that read them run."""
    a, b = devices["bf16"], pa.HIP16(0, storage="bf16")
    rng = np.random.default_rng(9)
    q, k, v = draw(rng, "bf16", 4, 1, 8, 128), draw(rng, "bf16", 4, 3000, 2, 128), draw(rng, "bf16", 4, 3000, 2, 128)
    lens = ((3000, 1200, 7, 2999), (1, 3000, 2048, 256))
    want = [Attention(q, k, v, places(4, 1, 3000, (1,) * 4, n), True, 0.1, "bf16") for n in lens]
    t = [[tensor(d, x) for x in (q, k, v)] for d in (a, b)]
    out = []
    for _ in range(8):
        for d, n, x in ((a, lens[0], t[0]), (b, lens[1], t[1])):
            out.append(d.attention_fw(*x, True, 0.1, d.new_sequences((1,) * 4, n)))
    for i, y in enumerate(out):
        check("y", y.to_vector(), want[i % 2].y, want[i % 2].tol_y)
    b.close()


def test_keys_behind_4_gib():
    """A cache whose last tokens lie more than 2^32 bytes behind its first."""
    dev = pa.HIP16(0, storage="bf16")
    tokens, d, hk = 4_300_000, 128, 4     # 4.4 GB of keys, the same of values
    k, v = (dev.new_tensor_by_constant(S([d, hk, tokens]), 0) for _ in range(2))
    rng = np.random.default_rng(10)
    n = 300
    q, ks, vs = draw(rng, "bf16", 1, 2, 8, d), draw(rng, "bf16", 1, n, hk, d), draw(rng, "bf16", 1, n, hk, d)
    for big, small in ((k, ks), (v, vs)):
        t = tensor(dev, small)
        _lib.call("phip_memcpy_d2d", dev.ctx(), big.handle() + 2 * d * hk * (tokens - n), t.handle(), 2 * small.size)
    tq = tensor(dev, q)
    # the keys before are zeros: score 0, value 0
    y = dev.attention_fw(tq, k, v, True, 1.0).to_vector().reshape(2, 8, d)
    for i in range(2):
        for h in range(8):
            m = n - 1 + i
            s = ks[0, :m, h // 2].astype(np.float64) @ q[0, i, h]
            p = np.exp(s - s.max())
            want = p @ vs[0, :m, h // 2] / (p.sum() + (tokens - n) * np.exp(-s.max()))
            # as in sequence_reference: products and sums of scores of up to 12 sigma, one rounding of p and of y
            size = np.abs(ks[0, :m, h // 2]) @ np.abs(q[0, i, h])
            rel = 2 * ((d + 8) * size.max() * 2.0 ** -24 + 2.0 ** -19) + 2.0 ** -8
            tol = 1.05 * (rel * (p @ np.abs(vs[0, :m, h // 2])) / (p.sum() + (tokens - n) * np.exp(-s.max())) + 2.0 ** -8 * np.abs(want)) + 1e-30
            check("y %d %d" % (i, h), y[i, h], want, tol)
    del k, v, tq, t
    dev.close()


@pytest.mark.parametrize("kind", KINDS)
def test_layer_together(devices, kind):
    """Norm, rotation and attention one after another, forward and back, as a layer runs them; its result and gradients
    against the plain forms fed with the device's own intermediate tensors, and against differences through the device."""
    dev = devices[kind]
    rng = np.random.default_rng(11)
    lens = (37, 1, 20)
    x = {"q": draw(rng, kind, 1, 60, 4, 64), "k": draw(rng, kind, 1, 60, 2, 64)}
    w = {n: rounded(1 + 0.1 * rng.standard_normal(64), kind) for n in x}
    v, gy = draw(rng, kind, 1, 60, 2, 64), draw(rng, kind, 1, 60, 4, 64)
    seqs, freqs = places(1, 60, 60, lens, None, True), pa.rotary_frequencies(32)[0]
    lists = dev.new_sequences(lens, packed=True)
    tx, tw = {n: tensor(dev, x[n]) for n in x}, {n: tensor(dev, w[n]) for n in w}
    tv, tg = tensor(dev, v), tensor(dev, gy)
    zeros = lambda t: dev.new_tensor_by_constant(t.shape(), 0)  # noqa: E731
    rq, rk = dev.norm_rotary_fw(tx["q"], tx["k"], tw["q"], tw["k"], freqs, 1e-6, seqs=lists)
    y, stats = dev.attention_fw(rq, rk, tv, True, 0.125, lists, stats=True)
    gq, gk, gv = zeros(rq), zeros(rk), zeros(tv)
    dev.attention_bw(rq, rk, tv, y, tg, stats, True, 0.125, lists, gq, gk, gv)
    gxq, gxk, gwq, gwk = zeros(rq), zeros(rk), zeros(tw["q"]), zeros(tw["k"])
    dev.norm_rotary_bw(tx["q"], tx["k"], tw["q"], tw["k"], gq, gk, freqs, 1e-6, False, 0, 1.0, lists, gxq, gxk, gwq, gwk)
    as_array = lambda t, like: t.to_vector().reshape(like.shape)  # noqa: E731
    a = Attention(as_array(rq, x["q"]), as_array(rk, x["k"]), v, seqs, True, 0.125, kind, gy)
    for name, t in (("y", y), ("gq", gq), ("gk", gk), ("gv", gv)):
        check(name, t.to_vector(), getattr(a, name), getattr(a, "tol_" + name))
    for n, r, g, gx, gw in (("q", rq, gq, gxq, gwq), ("k", rk, gk, gxk, gwk)):
        e = Rotary(x[n], seqs, freqs, kind, w=w[n], eps=1e-6, gy=as_array(g, x[n]))
        check("r" + n, r.to_vector(), e.y, e.tol_y)
        check("gx" + n, gx.to_vector(), e.gx, e.tol_gx)
        check("gw" + n, gw.to_vector(), e.gw, e.tol_gw)
    if kind != "f32":
        return
    # the sum of gy * y along a direction, by differences: the forward pass is off by about 2^-21 of the sum of |gy y| (a
    # few thousand terms of order 1, errors of either sign), over a step of 2^-7 twice; third derivatives leave 2^-14
    def loss(step, n, way):
        t = {m: tensor(dev, (x[m] + (step * way if m == n else 0)).astype(np.float32)) for m in x}
        p, r = dev.norm_rotary_fw(t["q"], t["k"], tw["q"], tw["k"], freqs, 1e-6, seqs=lists)
        return float((dev.attention_fw(p, r, tv, True, 0.125, lists).to_vector().astype(np.float64) * gy.reshape(-1)).sum())
    for n, g in (("q", gxq), ("k", gxk)):
        way = rng.standard_normal(x[n].shape)
        step = 2.0 ** -7
        got = (loss(step, n, way) - loss(-step, n, way)) / (2 * step)
        exact = float((g.to_vector().astype(np.float64) * way.reshape(-1)).sum())
        norm = float(np.sqrt((g.to_vector().astype(np.float64) ** 2).sum()))
        assert abs(got - exact) < 0.02 * norm + 2.0 ** -21 * np.abs(gy).sum() * 2 ** 6
