"""The operators of a self-attention layer between its projections, measured: rotary positions, the norm of each head
with the rotation in the same pass, and attention.

A case says which operator, whether it is a forward call or a training step (forward, then the gradients), the storage
type, the heads, and the sequences: "queries" and "keys" list their lengths.  "whole": samples of one length; "padded":
samples of the longest length (keys: of `capacity`, as in a cache) of which each uses its own part; "packed": one
sample with the sequences one after another.  Tensors are [size, heads, tokens] x batch with the first index fastest.
"""
import ctypes
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _same(length, n):
    return ",".join([str(length)] * n)


def listed():
    return [
        # one new token of one stream of 8 heads x 64 (a hidden size of 512): only latency counts
        dict(name="rotary_one_token", op="rotary", train=False, type="bf16", size=64, heads=8, kv_heads=8, pairs=32,
             interleaved=False, layout="padded", queries="1", keys="1234"),
        # the prompts of a batch of four, long contexts' last quarter of the positions, pairs side by side
        dict(name="rotary_prompt", op="rotary", train=False, type="f16", size=128, heads=32, kv_heads=8, pairs=64,
             interleaved=True, layout="padded", queries=_same(4096, 4), keys="16384,9000,4096,12288"),
        # training with a hidden size of 650 as 10 heads x 65, 64 samples of 35 words, half of a head rotated
        dict(name="rotary_train_odd", op="rotary", train=True, type="f32", size=65, heads=10, kv_heads=10, pairs=16,
             interleaved=False, layout="whole", queries=_same(35, 64), keys=_same(35, 64)),
        # a token for each of 64 streams at their own positions
        dict(name="norm_rotary_tokens", op="norm_rotary", train=False, type="bf16", size=128, heads=32, kv_heads=8,
             pairs=64, interleaved=False, layout="padded", queries=_same(1, 64),
             keys=",".join(str(17 + 613 * i % 30011) for i in range(64))),
        # prompts of very different lengths, packed
        dict(name="norm_rotary_prompt", op="norm_rotary", train=False, type="bf16", size=128, heads=32, kv_heads=8,
             pairs=64, interleaved=False, layout="packed", queries="7001,1,2049,513,6820", keys="7001,1,2049,513,6820"),
        # a training step on 16 samples of 1024 tokens
        dict(name="norm_rotary_train", op="norm_rotary", train=True, type="f16", size=64, heads=16, kv_heads=4, pairs=32,
             interleaved=True, layout="whole", queries=_same(1024, 16), keys=_same(1024, 16)),
        # a token for each of 16 streams against its cache
        dict(name="attention_tokens", op="attention", train=False, type="bf16", size=128, heads=32, kv_heads=8,
             causal=True, layout="padded", queries=_same(1, 16), capacity=8192,
             keys="8192,5,4097,1,7777,2048,6000,333,8191,64,1500,3001,129,7000,640,4444"),
        # one token against a very long cache
        dict(name="attention_long_cache", op="attention", train=False, type="f16", size=128, heads=32, kv_heads=8,
             causal=True, layout="padded", queries="1", capacity=131072, keys="130001"),
        # prompts of very different lengths, packed
        dict(name="attention_prompt", op="attention", train=False, type="bf16", size=128, heads=32, kv_heads=8,
             causal=True, layout="packed", queries="7001,1,2049,513,6820", keys="7001,1,2049,513,6820"),
        # a training step on two long samples with grouped heads
        dict(name="attention_train_long", op="attention", train=True, type="bf16", size=128, heads=32, kv_heads=8,
             causal=True, layout="whole", queries=_same(8192, 2), keys=_same(8192, 2)),
        # a training step of an encoder of heads of 64, padded samples
        dict(name="attention_train_padded", op="attention", train=True, type="f16", size=64, heads=16, kv_heads=16,
             causal=False, layout="padded", queries="1024,1000,777,1,64,512,900,1023", capacity=1024,
             keys="1024,1000,777,1,64,512,900,1023"),
        # a training step in 32 bits with a hidden size of 650 as 10 heads x 65, 64 samples of 35 words
        dict(name="attention_train_odd", op="attention", train=True, type="f32", size=65, heads=10, kv_heads=10,
             causal=True, layout="whole", queries=_same(35, 64), keys=_same(35, 64)),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm_rotary", "attention", "attention"])
    kv = rng.choice([1, 2, 4, 8, 10])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    size = rng.choice([16, 32, 64, 64, 65, 80, 96, 100, 128, 128])
    case = dict(op=op, type=rng.choice(["f32", "f16", "bf16"]), size=size, heads=heads, kv_heads=kv)
    if op == "attention":
        tokens = rng.random() < 0.35
        case.update(train=not tokens and rng.random() < 0.6, causal=tokens or rng.random() < 0.7)
        most = 4096 if case["type"] == "f32" else 8192
        if tokens:  # a few new tokens against caches
            n, new = _spread(rng, 1, 48), rng.choice([1, 1, 1, 2, 5])
            capacity = max(new, min(_spread(rng, 64, 65536), 400_000_000 // (n * kv * size * 4)))
            keys = [rng.randint(new, capacity) for _ in range(n)]
            case.update(layout="padded", queries=_same(new, n), keys=",".join(map(str, keys)), capacity=capacity)
            return case
        total = _spread(rng, 40, most)
        layout = rng.choice(["whole", "padded", "packed"])
        n = _spread(rng, 1, max(1, min(32, total // 8)))
        longest = max(1, total // n)
        if layout == "whole":
            lens = [longest] * n
        elif layout == "padded":
            lens = [rng.randint(0 if i else longest, longest) for i in range(n)]
        else:
            lens = [rng.randint(1, 2 * longest) for _ in range(n)]
        keys = lens
        if rng.random() < 0.3 and layout != "packed":  # other keys than queries
            longer = _spread(rng, longest, 2 * longest + 1)
            keys = [longer] * n if layout == "whole" else [min(longer, x + rng.randint(0, longer)) for x in lens]
        case.update(layout=layout, queries=",".join(map(str, lens)), keys=",".join(map(str, keys)), capacity=max(keys))
        return case
    pairs = rng.choice([size // 2, size // 2, size // 4])  # the whole head, or half of it
    case.update(train=rng.random() < 0.5, pairs=pairs, interleaved=rng.random() < 0.5)
    total = min(_spread(rng, 1, 20000), 60_000_000 // ((heads + kv) * size))
    layout = rng.choice(["whole", "padded", "packed"])
    n = _spread(rng, 1, max(1, min(64, total)))
    longest = max(1, total // n)
    if layout == "whole":
        lens = [longest] * n
    else:
        lens = [rng.randint(0 if i else longest, longest) for i in range(n)]
    keys = lens if layout == "whole" else [x + rng.randint(0, 100000) for x in lens]
    case.update(layout=layout, queries=",".join(map(str, lens)), keys=",".join(map(str, keys)))
    return case


def _extents(case):
    """(query lengths, key lengths, tokens of a sample: queries, keys, batch)."""
    lq, lk = _ints(case["queries"]), _ints(case["keys"])
    if case["layout"] == "packed":
        return lq, lk, sum(lq), sum(lk), 1
    return lq, lk, max(lq), case.get("capacity", max(lk)), len(lq)


def _frequencies(pairs):
    return np.asarray([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=np.float32)


def prepare(case, seed):
    dtype = _TYPES[case["type"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lq, lk, tq, tk, bs = _extents(case)

    def normal(*shape):
        x = torch.empty(shape, dtype=dtype, device="cuda")
        flat, step = x.view(-1), 1 << 26
        for at in range(0, flat.numel(), step):
            n = min(step, flat.numel() - at)
            flat[at:at + n] = torch.randn(n, generator=gen, device="cuda")
        return x

    d, hq, hk = case["size"], case["heads"], case["kv_heads"]
    s = dict(case=case, lq=lq, lk=lk)
    if case["op"] == "attention":
        s["q"], s["k"], s["v"] = normal(bs, tq, hq, d), normal(bs, tk, hk, d), normal(bs, tk, hk, d)
        if case["train"]:
            s["gy"] = normal(bs, tq, hq, d)
        s["scale"] = 1.0 / math.sqrt(d)
    else:
        s["q"], s["k"] = normal(bs, tq, hq, d), normal(bs, tq, hk, d)
        if case["train"]:
            s["gq"], s["gk"] = normal(bs, tq, hq, d), normal(bs, tq, hk, d)
        if case["op"] == "norm_rotary":
            s["wq"], s["wk"] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
            s["eps"] = 1e-6
        s["f"] = _frequencies(case["pairs"])
        s["angles"] = torch.tensor(s["f"], device="cuda", dtype=torch.float64)
    if own:
        _prepare_own(s, tq, tk, bs)
    return s


def _places(s):
    """Where each sequence lies: (sample, first query row, queries, first key row, keys)."""
    at_q = at_k = 0
    for i, (n, m) in enumerate(zip(s["lq"], s["lk"])):
        if s["case"]["layout"] == "packed":
            yield 0, at_q, n, at_k, m
            at_q, at_k = at_q + n, at_k + m
        else:
            yield i, 0, n, 0, m


# ---- plain forms: elementary operations in 32 bits ------------------------------------------------------------------


def _angles(s):
    """cos and sin for each token, [batch, tokens, 1, pairs]; the angle itself needs 64 bits at far positions."""
    q = s["q"]
    if s["case"]["layout"] == "whole":
        at = torch.arange(q.shape[1], device=q.device).expand(q.shape[0], -1)
    else:
        at = torch.zeros(q.shape[0], q.shape[1], dtype=torch.int64, device=q.device)
        for b, a, n, _, m in _places(s):
            at[b, a:a + n] = torch.arange(m - n, m, device=q.device)
    angle = at[:, :, None, None].double() * s["angles"]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _turn(x, cos, sin, pairs, interleaved):
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return y


def _used(s, x):
    """Rows that no sequence covers are zero."""
    if s["case"]["layout"] == "padded":
        for b, _, n, _, _ in _places(s):
            x[b, n:] = 0
    return x


def _plain_rotary(s):
    case = s["case"]
    cos, sin = _angles(s)
    out, eps = {}, s.get("eps")
    for name in ("q", "k"):
        x = s[name].float()
        if eps is None:
            n = x
        else:
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
            w = s["w" + name].float()
            n = x * r * w
        out["y" + name] = _used(s, _turn(n, cos, sin, case["pairs"], case["interleaved"])).to(s[name].dtype)
        if case["train"]:
            gy = _used(s, s["g" + name].float())
            g = _turn(gy, cos, -sin, case["pairs"], case["interleaved"])
            if eps is not None:
                out["gw" + name] = (g * x * r).sum((0, 1, 2)).to(s[name].dtype)
                gw = g * w
                g = r * (gw - x * r * r * (gw * x).mean(-1, keepdim=True))
            out["gx" + name] = g.to(s[name].dtype)
    return out


def _plain_attention_part(q, k, v, scale, causal, gy=None):
    """q [n, rows, tokens, d], k and v [n, keys, d] (n groups of heads): y and, with gy, the gradients."""
    n, g, lq, d = q.shape
    lk = k.shape[1]
    flat = q.reshape(n, g * lq, d)
    s = torch.matmul(flat, k.transpose(1, 2).contiguous()).view(n, g, lq, lk) * scale
    if causal:
        hidden = torch.arange(lk, device=q.device)[None, :] > torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        s = s.masked_fill(hidden, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    del s
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    pf = p.view(n, g * lq, lk)
    y = torch.matmul(pf, v).view(n, g, lq, d)
    if gy is None:
        return y, None, None, None
    gyf = gy.reshape(n, g * lq, d)
    gv = torch.matmul(pf.transpose(1, 2).contiguous(), gyf)
    dp = torch.matmul(gyf, v.transpose(1, 2).contiguous()).view(n, g, lq, lk)
    ds = p * (dp - (gy * y).sum(-1, keepdim=True)) * scale
    del dp
    dsf = ds.view(n, g * lq, lk)
    return y, torch.matmul(dsf, k).view(n, g, lq, d), torch.matmul(dsf.transpose(1, 2).contiguous(), flat), gv


def _plain_attention(s):
    case = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    bs, tq, hq, d = q.shape
    hk, train = k.shape[2], case["train"]
    g = hq // hk
    out = dict(y=torch.zeros_like(q))
    if train:
        out.update(gq=torch.zeros_like(q), gk=torch.zeros_like(k), gv=torch.zeros_like(v))
    if case["layout"] == "whole":  # all samples in one go
        parts = [(slice(0, bs), slice(0, tq), slice(0, k.shape[1]))]
    else:
        parts = [(slice(b, b + 1), slice(a, a + n), slice(c, c + m)) for b, a, n, c, m in _places(s) if n and m]
    for b, rq, rk in parts:
        def heads_first(x, rows, rep):  # [samples * kv heads, (heads of a group,) tokens, d] in 32 bits
            x = x[b, rows]
            x = x.reshape(x.shape[0], x.shape[1], hk, rep, d).permute(0, 2, 3, 1, 4).float()
            return x.reshape(-1, rep, x.shape[3], d)
        qs, ks, vs = heads_first(q, rq, g), heads_first(k, rk, 1)[:, 0], heads_first(v, rk, 1)[:, 0]
        gs = heads_first(s["gy"], rq, g) if train else None
        step = max(1, (1 << 28) // (g * qs.shape[2] * ks.shape[1]))
        done = [_plain_attention_part(qs[i:i + step], ks[i:i + step], vs[i:i + step], s["scale"], case["causal"],
                                      gs[i:i + step] if train else None) for i in range(0, qs.shape[0], step)]
        for at, (name, rows, rep) in enumerate((("y", rq, g), ("gq", rq, g), ("gk", rk, 1), ("gv", rk, 1))):
            if name in out:
                x = torch.cat([z[at] for z in done])
                x = x.reshape(b.stop - b.start, hk, rep, -1, d).permute(0, 3, 1, 2, 4)
                out[name][b, rows] = x.reshape(x.shape[0], x.shape[1], hk * rep, d).to(q.dtype)
    return out


# ---- the framework's calls ------------------------------------------------------------------------------------------

_devices = {}


def _device(kind):
    """One device object per storage type, as a program has it."""
    import primitiv_amd
    if kind not in _devices:
        _devices[kind] = primitiv_amd.HIP(0) if kind == "f32" else primitiv_amd.HIP16(0, storage=kind)
    return _devices[kind]


def _prepare_own(s, tq, tk, bs):
    """The device, the sequences of the batch (made once, used by every layer) and the memory of the results."""
    from primitiv_amd import _lib
    case = s["case"]
    kind = case["type"]
    dev = s["dev"] = _device(kind)
    s["seqs"] = None if case["layout"] == "whole" else dev.new_sequences(s["lq"], s["lk"], packed=case["layout"] == "packed")
    handle = s["seqs"].handle() if s["seqs"] is not None else None
    d, hq, hk = case["size"], case["heads"], case["kv_heads"]

    def like(*names):
        return [torch.empty_like(s[n]) for n in names]

    def at(*tensors):
        return [t.data_ptr() for t in tensors]

    fn = getattr(_lib.lib(), "phip_%s_fw_%s" % (case["op"], kind))
    fill = getattr(_lib.lib(), "phip_fill_" + kind)
    train = case["train"]
    calls = s["calls"] = []
    ctx = dev.ctx()
    if case["op"] == "attention":
        s["out"] = dict(zip(("y", "gq", "gk", "gv") if train else ("y",), like("q", "q", "k", "v")))
        s["stats"] = torch.empty(bs * tq * hq, dtype=torch.float32, device="cuda") if train else None
        stats = s["stats"].data_ptr() if train else None
        shape = (d, hq, hk, tq, tk, bs, handle, int(case["causal"]), s["scale"])
        calls.append((fn, (ctx, *at(s["q"], s["k"], s["v"], s["out"]["y"]), stats, *shape)))
        if train:
            grads = [s["out"][n] for n in ("gq", "gk", "gv")]
            calls += [(fill, (ctx, g.data_ptr(), 0.0, g.numel())) for g in grads]
            calls.append((getattr(_lib.lib(), "phip_attention_bw_" + kind),
                          (ctx, *at(s["q"], s["k"], s["v"], s["out"]["y"]), stats, *at(s["gy"], *grads), *shape)))
    else:
        norm = case["op"] == "norm_rotary"
        weights = at(s["wq"], s["wk"]) if norm else []
        s["f_held"] = np.ascontiguousarray(s["f"])
        f = s["f_held"].ctypes.data_as(ctypes.POINTER(ctypes.c_float))
        shape = (d, hq, hk, tq, bs, handle, 0, f, case["pairs"], int(case["interleaved"]), 1.0)
        shape += (s["eps"],) if norm else ()
        s["out"] = dict(zip(("yq", "yk"), like("q", "k")))
        calls.append((fn, (ctx, *at(s["q"], s["k"]), *weights, *at(s["out"]["yq"], s["out"]["yk"]), *shape)))
        if train:
            names = ("gxq", "gxk", "gwq", "gwk") if norm else ("gxq", "gxk")
            s["out"].update(zip(names, like("q", "k", *(("wq", "wk") if norm else ()))))
            grads = [s["out"][n] for n in names]
            calls += [(fill, (ctx, g.data_ptr(), 0.0, g.numel())) for g in grads]
            read = at(s["q"], s["k"]) if norm else []
            calls.append((getattr(_lib.lib(), "phip_%s_bw_%s" % (case["op"], kind)),
                          (ctx, *read, *weights, *at(s["gq"], s["gk"]), *at(*grads), *shape)))
    torch.cuda.synchronize()  # the inputs are there before another stream reads them


def _run_own(s):
    """The calls through the C ABI: the framework's kernels run on the device's own stream, in order."""
    from primitiv_amd import _lib
    for fn, args in s["calls"]:
        _lib.check(fn(*args))
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    if state["case"]["op"] == "attention":
        return _plain_attention(state)
    return _plain_rotary(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    lq, lk, tq, _, bs = _extents(case)
    d, hq, hk = case["size"], case["heads"], case["kv_heads"]
    item = 4 if case["type"] == "f32" else 2
    if case["op"] == "attention":
        pairs = 0
        for n, m in zip(lq, lk):
            if case["causal"]:  # query i sees keys 0 .. i + m - n
                first = max(0, n - m)  # queries before it see nothing
                pairs += (n - first) * ((first + m - n + 1) + m) // 2
            else:
                pairs += n * m
        rows = d * (hq * sum(lq)), d * (hk * sum(lk))
        moved = 2 * rows[0] + 2 * rows[1]  # q, k, v in, y out
        if case["train"]:
            moved += 2 * rows[0] + 2 * rows[1]  # gy in, gq, gk, gv out
        return dict(bytes=item * moved, flops=(14 if case["train"] else 4) * d * pairs * hq)
    rows = d * (hq + hk) * sum(lq)
    per = 4 * rows if case["train"] else 2 * rows  # x and y, gy and gx
    norm = case["op"] == "norm_rotary"
    return dict(bytes=item * per, flops=rows * ((20 if norm else 6) if case["train"] else (7 if norm else 3)))


# ---- the definition in 64 bits --------------------------------------------------------------------------------------


def _exact_turned(x, first, case):
    """Rows x [tokens, heads, size] in 64 bits at positions first, first + 1, ...: each pair times a complex number."""
    pairs = case["pairs"]
    f = torch.tensor(_frequencies(pairs).astype(np.float64), device=x.device)
    at = torch.arange(x.shape[0], device=x.device, dtype=torch.float64) + first
    turn = torch.polar(torch.ones(x.shape[0], pairs, dtype=torch.float64, device=x.device), at[:, None] * f)[:, None]
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], pairs, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(head.shape)
    else:
        z = torch.complex(head[..., :pairs].contiguous(), head[..., pairs:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, rest], -1)


def exact(case, seed):
    if case["op"] == "attention" and work(case)["flops"] > 4e13:
        return None
    s = prepare(case, seed)
    train = case["train"]
    wide = torch.float64
    out = {}
    if case["op"] != "attention":
        for name in ("q", "k"):
            x = s[name].to(wide).requires_grad_(train)
            w = s["w" + name].to(wide).requires_grad_(train) if "eps" in s else None
            y = torch.zeros_like(s[name], dtype=wide)
            total = 0
            for b, a, n, _, m in _places(s):
                rows = x[b, a:a + n]
                if w is not None:
                    rows = rows / torch.sqrt((rows ** 2).sum(-1, keepdim=True) / case["size"] + s["eps"]) * w
                rows = _exact_turned(rows, m - n, case)
                y[b, a:a + n] = rows.detach()
                if train:
                    total = total + (rows * s["g" + name][b, a:a + n].to(wide)).sum()
            out["y" + name] = y
            if train:
                total.backward()
                out["gx" + name] = x.grad
                if w is not None:
                    out["gw" + name] = w.grad
        return out
    q, k, v = (s[n] for n in ("q", "k", "v"))
    g = q.shape[2] // k.shape[2]
    out["y"] = torch.zeros_like(q, dtype=wide)
    if train:
        out.update(gq=torch.zeros_like(q, dtype=wide), gk=torch.zeros_like(k, dtype=wide), gv=torch.zeros_like(v, dtype=wide))
    for b, a, n, c, m in _places(s):
        if n == 0 or m == 0:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if case["causal"]:
            seen = torch.tril(seen, diagonal=m - n)
        empty = ~seen.any(1)
        for h in range(q.shape[2]):
            one = [t.to(wide).requires_grad_(train) for t in (q[b, a:a + n, h], k[b, c:c + m, h // g], v[b, c:c + m, h // g])]
            score = (one[0] * s["scale"]) @ one[1].T
            score = torch.where(seen | empty[:, None], score, torch.full((), -math.inf, dtype=wide, device=q.device))
            y = torch.where(empty[:, None], 0.0, torch.softmax(score, 1) @ one[2])
            out["y"][b, a:a + n, h] = y.detach()
            if train:
                y.backward(s["gy"][b, a:a + n, h].to(wide))
                out["gq"][b, a:a + n, h] = one[0].grad
                out["gk"][b, c:c + m, h // g] += one[1].grad
                out["gv"][b, c:c + m, h // g] += one[2].grad
    return out
