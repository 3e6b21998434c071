"""Chunks of new tokens over a paged cache (tle_append_paged,
tle_append_bf16_paged, tle_prefill_bf16_paged) against the formulas in 64 bits.

Tolerances, per value (u = half a step of a type, relative: bf16 2^-8, fp32
2^-24):
* append: the angle is the 32-bit number fl32(pos * f_i) by definition; sine
  and cosine are off by 2 ulp (2^-23) at most, the two products and their sum
  by a rounding each, so a rotated element is within (|a| + |b|) 2^-22 of the
  formula, plus u of the stored type.
* attend: a score is a sum of 64 products in 32 bits: off by at most
  ds = 2^-17 sum|q k| / 8 with the tensor cores' truncating sums; a weight is
  then off by 2 (ds + |s| 2^-23 + 2^-22) relative (numerator and sum), and the
  sum over rows adds (rows / 16 + 16) 2^-23; with bf16 activations a weight is
  rounded to bf16 (2^-8) after an exponential good to 2^-13.  All of it times
  sum w |v|; the result is rounded once to the type of q.
"""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tinyllama-engine_b200"))

pytestmark = pytest.mark.gpu

HD, BASE = 64, 10000.0
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}


def dtype(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16}[name]


class Case:
    """A paged cache of random rows and a batch over it, on the GPU."""

    def __init__(self, pos, new, heads=(32, 4), page=64, act="f32", pool="bf16", layers=2, seed=0, spare=3,
                 pad=0, max_ctas=0, scale=1.0):
        import torch
        import tle
        self.pos, self.new, self.heads, self.page, self.act = list(pos), list(new), heads, page, act
        self.H, self.KH = heads
        self.layers, self.layer = layers, layers - 1
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-(p + m) // page) for p, m in zip(pos, new)]
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        self.tables, at = [], 0
        for k in need:
            self.tables.append(ids[at:at + k].clone())
            at += k
        self.free = ids[at:]
        shape = tle.Shape(layers, self.H, self.KH, HD, BASE)
        self.cache = tle.PagedKVCache(n_pages, page, shape, dtype=dtype(pool))
        self.cache.key_pool.copy_(torch.randn(self.cache.key_pool.shape, generator=g, device="cuda"))
        self.cache.value_pool.copy_(torch.randn(self.cache.value_pool.shape, generator=g, device="cuda"))
        T = sum(new)
        rnd = lambda w: torch.randn(T + pad, w * HD, generator=g, device="cuda").to(dtype(act))  # noqa: E731
        self.T = T
        self.q, self.k, self.v = rnd(self.H) * scale, rnd(self.KH), rnd(self.KH)
        self.out = torch.full_like(self.q, 7.0)
        self.batch = tle.PagedChunkBatch(self.cache, self.tables, pos, new, max_ctas=max_ctas)

    def positions(self):
        return np.concatenate([np.arange(p, p + m) for p, m in zip(self.pos, self.new)] or [[]]).astype(np.int64)

    def flat_rows(self, s, rows):
        """Rows of sequence s as rows of a layer's flattened pool."""
        t = self.tables[s].cpu().numpy().astype(np.int64)
        return t[rows // self.page] * self.page + rows % self.page


def angles(positions):
    f = (np.float32(1) / np.power(BASE, np.arange(0, HD, 2) / HD).astype(np.float32)).astype(np.float32)
    return (positions.astype(np.float32)[:, None] * f).astype(np.float64)


def rotated(x, positions):
    """64-bit rotation of x [tokens][heads * 64], and |a| + |b| of each element's pair."""
    y = x.double().cpu().numpy().reshape(len(positions), -1, HD // 2, 2)
    a = angles(positions)[:, None, :]
    z = np.stack([y[..., 0] * np.cos(a) - y[..., 1] * np.sin(a), y[..., 0] * np.sin(a) + y[..., 1] * np.cos(a)], -1)
    size = np.repeat(np.abs(y).sum(-1, keepdims=True), 2, -1)
    return z.reshape(x.shape), size.reshape(x.shape)


def attention64(c, q):
    """The formula in 64 bits: results and tolerances [T][H * 64]."""
    import torch
    out = torch.zeros(c.T, c.H * HD, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    G = c.H // c.KH
    t0 = 0
    for s, (p, m) in enumerate(zip(c.pos, c.new)):
        if m == 0:
            continue
        rows = torch.from_numpy(c.flat_rows(s, np.arange(p + m))).cuda()
        for h in range(c.H):
            sl = slice((h // G) * HD, (h // G + 1) * HD)
            k = c.cache.key_pool[c.layer].view(-1, c.KH * HD)[rows, sl].double()
            v = c.cache.value_pool[c.layer].view(-1, c.KH * HD)[rows, sl].double()
            qq = q[t0:t0 + m, h * HD:(h + 1) * HD].double()
            e = qq @ k.T / 8
            hide = torch.arange(p + m, device="cuda")[None, :] > p + torch.arange(m, device="cuda")[:, None]
            big = (qq.abs() @ k.abs().T / 8).masked_fill(hide, 0).amax(1, keepdim=True)
            top = e.abs().masked_fill(hide, 0).amax(1, keepdim=True)
            w = torch.softmax(e.masked_fill(hide, -float("inf")), 1)
            o = w @ torch.where(hide.all(0)[:, None], torch.zeros_like(v), v)
            size = w @ v.abs()
            rel = 2 * (big * 2.0 ** -17 + top * 2.0 ** -23 + 2.0 ** -22) + ((p + m) / 16 + 16) * 2.0 ** -23
            if c.act == "bf16":
                rel = rel + 2.0 ** -8 + 2.0 ** -12
            out[t0:t0 + m, h * HD:(h + 1) * HD] = o
            tol[t0:t0 + m, h * HD:(h + 1) * HD] = rel * size + U[c.act] * (o.abs() + rel * size)
        t0 += m
    return out, tol


def check_attend(c, q=None, out=None):
    import torch
    import tle
    q = c.q if q is None else q
    out = c.out if out is None else out
    c.batch.attend(q, out, c.layer)
    torch.cuda.synchronize()
    want, tol = attention64(c, q)
    d = (out[:c.T].double() - want).abs()
    assert bool((d <= tol).all()), float((d / tol).max())
    assert tle.device_error() == 0


CASES = [
    dict(pos=[0], new=[1]),                                             # one token, one row
    dict(pos=[0], new=[129]),
    dict(pos=[126, 127, 128, 129], new=[1, 1, 1, 1]),                   # around a tile's edge
    dict(pos=[63, 64, 0, 500], new=[1, 2, 3, 0]),                       # a sequence without tokens
    dict(pos=[0, 0, 7], new=[0, 0, 5]),
    dict(pos=[300], new=[16]), dict(pos=[300], new=[17]),               # around the row tiles (8 heads a token)
    dict(pos=[300], new=[32]), dict(pos=[300], new=[33]),
    dict(pos=[1000, 3, 250], new=[40, 257, 1], page=128),
    dict(pos=[2000, 1029, 1500, 2040], new=[1, 1, 1, 1], page=1024),
    dict(pos=[5000], new=[3]),                                          # one sequence over many CTAs
    dict(pos=[70, 131], new=[45, 130], heads=(8, 8)),                   # one query head per KV head
    dict(pos=[70, 131], new=[45, 130], heads=(12, 4)),                  # groups of 3, of 5, of 7
    dict(pos=[70, 131], new=[45, 130], heads=(20, 4), page=256),
    dict(pos=[70, 0], new=[1, 300], heads=(7, 1)),
    dict(pos=[64], new=[3], heads=(128, 1)),                            # a token fills a row tile
    dict(pos=list(range(0, 1600, 25)), new=[1 + i % 5 for i in range(64)]),
    dict(pos=[900, 10, 400], new=[100, 200, 300], max_ctas=3),          # several items per CTA
    dict(pos=[900, 10, 400], new=[100, 200, 300], max_ctas=1),
]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_attend_matches_the_formula(cuda, i, act):
    check_attend(Case(**CASES[i], act=act, seed=i))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attend_large_scores(cuda, act):
    """Weights concentrated on a few rows (scores up to about +-100)."""
    check_attend(Case([700, 130], [20, 1], act=act, scale=25.0, seed=3))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attend_falling_and_rising_scores(cuda, act):
    """Scores that grow along the rows (every tile moves the running maximum)
    and that fall (none after the first does)."""
    import torch
    for sign in (1.0, -1.0):
        c = Case([900], [2], act=act, seed=4)
        ramp = torch.linspace(-1, 1, 902, device="cuda") * sign
        rows = torch.from_numpy(c.flat_rows(0, np.arange(902))).cuda()
        kp = c.cache.key_pool[c.layer].view(-1, 256)
        c.q.abs_().mul_(3)
        kp[rows] = (ramp[:, None] * 6).expand(-1, 256).to(kp.dtype)
        check_attend(c)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([200], [3]), ([0, 60], [70, 1]), ([120], [150])])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_rows_nobody_attends_to_do_not_matter(cuda, act, pos, new, bad):
    """NaN and infinities behind a sequence's last row, in other pages, other
    layers: the results are those of finite rows, bit for bit."""
    import torch
    c = Case(pos, new, act=act, seed=5)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    for pool in (c.cache.key_pool, c.cache.value_pool):
        keep = torch.zeros(pool.shape[1] * pool.shape[2], dtype=torch.bool, device="cuda")
        for s, (p, m) in enumerate(zip(pos, new)):
            keep[torch.from_numpy(c.flat_rows(s, np.arange(p + m))).cuda()] = True
        pool[c.layer].view(-1, 256)[~keep] = float(bad)
        pool[:c.layer] = float(bad)
    check_attend(c)
    assert torch.equal(first, c.out)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,at", [([200], [3], 201), ([0], [70], 40), ([100], [300], 260), ([5], [1], 2),
                                        ([1000], [40], 1039), ([1000], [1], 1000), ([130], [33], 3)])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_bad_row_reaches_only_the_tokens_that_attend_to_it(cuda, act, pos, new, at, bad, where):
    import torch
    import tle
    c = Case(pos, new, act=act, seed=6)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    want, tol = attention64(c, c.q)
    row = int(c.flat_rows(0, np.array([at]))[0])
    pool = c.cache.key_pool if where == "k" else c.cache.value_pool
    pool[c.layer].view(-1, 256)[row, 64:128] = float(bad)      # KV head 1: query heads 8 .. 15
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    sees = torch.arange(new[0], device="cuda") + pos[0] >= at
    mine = slice(8 * HD, 16 * HD)
    assert bool(((c.out.double() - want).abs() <= tol)[~sees].all())
    assert torch.equal(c.out[:, :8 * HD], first[:, :8 * HD]) and torch.equal(c.out[:, 16 * HD:], first[:, 16 * HD:])
    hit = c.out[sees, mine]
    if where == "v":
        assert bool((~torch.isfinite(hit)).all())
    elif bad == "nan":
        assert bool(torch.isnan(hit).all())
    else:                       # a score of +-inf (or NaN): the row alone, or no weight at all
        now, _ = attention64(c, c.q)
        fine = torch.isfinite(now[sees, mine])
        assert bool(torch.isnan(hit[~fine]).all()) or bool((~torch.isfinite(hit[~fine])).all())
    assert tle.device_error() == 0


def test_attend_leaves_rows_behind_the_last_token(cuda):
    import torch
    c = Case([100, 20], [3, 4], pad=5)
    check_attend(c)
    assert bool((c.out[7:] == 7.0).all())


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attend_row_strides(cuda, act):
    """q inside a fused q/k/v buffer, out inside a wider one."""
    import torch
    c = Case([90, 300], [33, 2], act=act, seed=8)
    qkv = torch.randn(c.T, 40 * HD, device="cuda").to(c.q.dtype)
    wide = torch.full((c.T, 32 * HD + 24), 7.0, device="cuda", dtype=c.q.dtype)
    check_attend(c, q=qkv[:, :32 * HD], out=wide[:, 16:16 + 32 * HD])
    assert bool((wide[:, :16] == 7).all()) and bool((wide[:, 16 + 32 * HD:] == 7).all())


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_attend_is_reproducible_and_replays(cuda, act):
    """Same bits in a second call, on another stream, and from a captured
    graph after the inputs changed in place."""
    import torch
    c = Case([700, 50, 1300], [40, 9, 1], act=act, seed=9)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    c.out.fill_(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.batch.attend(c.q, c.out, c.layer, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, c.out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (c.q, c.k, c.v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = c.out.clone()
        c.batch.run(c.q, c.k, c.v, c.out, c.layer)
        torch.cuda.synchronize()
        assert torch.equal(got, c.out)


@pytest.mark.parametrize("pos,new", [([700, 50, 1300], [40, 9, 1]), ([5000, 20], [70, 2])])
def test_a_replay_under_another_plan_does_nothing(cuda, pos, new):
    """A captured call whose descriptor was replaced: 0x10b, and neither pools
    nor results change; under a plan with the same numbers it is right."""
    import torch
    import tle
    c = Case(pos, new, seed=13)
    c.batch.run(c.q, c.k, c.v, c.out, c.layer)          # the buffer of the rotated q
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    plan = bytes(c.batch.plan)
    c.batch.set_positions([p - 1 for p in pos], new)
    assert bytes(c.batch.plan) == plan
    graph.replay()
    torch.cuda.synchronize()
    got = c.out.clone()
    c.out.fill_(3)
    c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    torch.cuda.synchronize()
    assert torch.equal(got, c.out) and tle.device_error() == 0
    refused = 0
    for other in ([0] * len(pos), [p // 3 for p in pos]):
        c.batch.set_positions(other, new)
        pools = (c.cache.key_pool.clone(), c.cache.value_pool.clone())
        c.out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        if bytes(c.batch.plan) == plan:                 # the split may be the same there too
            got = c.out.clone()
            c.batch.run(c.q, c.k, c.v, c.out, c.layer)
            torch.cuda.synchronize()
            assert torch.equal(got, c.out) and tle.device_error() == 0
            continue
        refused += 1
        assert tle.device_error() == 0x10b
        assert bool((c.out == 3).all())
        assert torch.equal(pools[0], c.cache.key_pool) and torch.equal(pools[1], c.cache.value_pool)
    assert refused
    c.out.fill_(3)
    c.batch.set_positions(pos, [1] * len(pos))          # fewer tokens
    graph.replay()
    torch.cuda.synchronize()
    assert tle.device_error() == 0x10b and bool((c.out == 3).all())


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,bad", [([700, 50, 1300], [40, 9, 1], None), ([9000], [100], None), ([0, 4000], [600, 3], None),
                                         ([120, 40], [150, 3], 200)])
def test_attend_in_place(cuda, act, pos, new, bad):
    """out is q, with items cut over several CTAs and rows computed again."""
    import torch
    c = Case(pos, new, act=act, seed=14)
    if bad is not None:
        c.cache.value_pool.view(c.layers, -1, c.KH * HD)[c.layer, int(c.flat_rows(0, np.array([bad]))[0])] = float("inf")
    c.batch.attend(c.q, c.out, c.layer)
    c.batch.attend(c.q, c.q, c.layer)
    torch.cuda.synchronize()
    assert torch.equal(c.q.nan_to_num(9.0), c.out.nan_to_num(9.0))


@pytest.mark.parametrize("new", [1, 4, 64])
def test_long_fp32_sums_do_not_drift(cuda, new):
    """All rows of V positive, so that sums that are cut off instead of rounded
    drift.  Each of at most 48 MMAs between two rounded sums loses up to 2^-23
    of the sum, the 16000 / 256 rounded ones (16 pieces and 16 joins more) up to
    2^-24 each; a score is 12 MMAs' sum of |q k| / 8 off by 2^-23 each, its
    weight and their sum by that and by 2^-22 and |s| 2^-23."""
    import torch
    c = Case([16000], [new], heads=(8, 2), seed=15, scale=0.1)
    c.cache.value_pool.abs_()
    c.batch.attend(c.q, c.out, c.layer)
    want = torch.empty(new, c.H * HD, dtype=torch.float64, device="cuda")
    rows = torch.from_numpy(c.flat_rows(0, np.arange(16000 + new))).cuda()
    size = 0.0
    for h in range(c.H):
        sl = slice(h // 4 * HD, (h // 4 + 1) * HD)
        k = c.cache.key_pool[c.layer].view(-1, c.KH * HD)[rows, sl].double()
        v = c.cache.value_pool[c.layer].view(-1, c.KH * HD)[rows, sl].double()
        q = c.q[:, h * HD:(h + 1) * HD].double()
        hide = torch.arange(16000 + new, device="cuda")[None, :] > 16000 + torch.arange(new, device="cuda")[:, None]
        w = torch.softmax((q @ k.T / 8).masked_fill(hide, -float("inf")), 1)
        want[:, h * HD:(h + 1) * HD] = w @ v
        size = max(size, float((q.abs() @ k.abs().T / 8).max()))
    tol = 48 * 2.0 ** -23 + (16000 / 256 + 32) * 2.0 ** -24 + 2 * (12 * size * 2.0 ** -23 + 2.0 ** -22 + size * 2.0 ** -23)
    assert float(((c.out.double() - want).abs() / want).max()) <= tol


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_long_prompt_at_some_tokens(cuda, act):
    """20000 tokens at once (more blocks of rows than the plan sorts), some
    tokens of it against the formula; tolerance as above."""
    import torch
    import tle
    c = Case([37], [20000], act=act, seed=17, layers=1)
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    rows = torch.from_numpy(c.flat_rows(0, np.arange(20037))).cuda()
    at = torch.tensor([0, 1, 90, 91, 127, 128, 4095, 9999, 15000, 19998, 19999], device="cuda")
    hide = torch.arange(20037, device="cuda")[None, :] > 37 + at[:, None]
    u = U["bf16" if act == "bf16" else "f32"]
    for h in range(0, c.H, 5):
        sl = slice(h // 8 * HD, (h // 8 + 1) * HD)
        k = c.cache.key_pool[0].view(-1, c.KH * HD)[rows, sl].double()
        v = c.cache.value_pool[0].view(-1, c.KH * HD)[rows, sl].double()
        q = c.q[at, h * HD:(h + 1) * HD].double()
        e = (q @ k.T / 8).masked_fill(hide, -float("inf"))
        w = torch.softmax(e, 1)
        ds = 2.0 ** -17 * float((q.abs() @ k.abs().T / 8).max())
        rel = 2 * (ds + float(e[~hide].abs().max()) * 2.0 ** -23 + 2.0 ** -22) + (20037 / 16 + 16) * 2.0 ** -23
        rel += 2.0 ** -8 + 2.0 ** -13 if act == "bf16" else 0.0
        want = w @ v
        tol = rel * (w @ v.abs()) + u * (want.abs() + rel * (w @ v.abs()))
        assert bool(((c.out[at, h * HD:(h + 1) * HD].double() - want).abs() <= tol).all())
    assert tle.device_error() == 0


def test_tensors_are_checked(cuda):
    import torch
    import tle
    c = Case([100, 20], [3, 4])
    b, T = c.batch, c.T
    f = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")  # noqa: E731
    bf = torch.bfloat16
    for q, out in ((c.q.cpu(), c.out), (c.q, c.out.cpu()), (c.q.to(bf), c.out), (c.q, c.out.to(bf)), (c.q.double(), c.out.double()),
                   (c.q[:T - 1], c.out), (c.q, c.out[:T - 1]), (c.q[:, :-64], c.out), (f(2048, T).T, c.out), (c.q.flatten(), c.out)):
        with pytest.raises(ValueError):
            b.attend(q, out, 0)
    for q, out, layer in ((f(T, 2052)[:, :2048], c.out, 0), (c.q, f(1, 2048).expand(T, 2048), 0), (c.q, c.out, 2), (c.q, c.out, -1),
                          (f(T * 2048 + 2)[2:].view(T, 2048), c.out, 0), (c.q, f(T * 2048 + 1)[1:].view(T, 2048), 0)):
        with pytest.raises(tle.TleError):
            b.attend(q, out, layer)
    for q, k, v, qo in ((c.q, c.k, c.v, None), (None, c.k, c.v, c.q), (c.q, c.k, c.v.to(bf), c.q), (c.q, c.k[:, :-64], c.v, c.q),
                        (c.q, c.k, c.v, f(T, 2112)[:, :2048]), (c.q.to(bf), c.k, c.v, c.q)):
        with pytest.raises(ValueError):
            b.append(q, k, v, 0, q_out=qo)
    plain = tle.PagedKVCache(8, 64, c.cache.shape)
    with pytest.raises(ValueError):
        tle.PagedChunkBatch(plain, c.tables, [0, 0], [1, 1]).attend(c.q, c.out, 0)
    with pytest.raises(ValueError):
        tle.PagedChunkBatch(plain, [t.long() for t in c.tables], [0, 0], [1, 1])
    with pytest.raises(ValueError):
        tle.PagedChunkBatch(plain, [t.cpu() for t in c.tables], [0, 0], [1, 1])
    with pytest.raises(ValueError):
        tle.PagedChunkBatch(plain, c.tables, [0], [1, 1])
    with pytest.raises(tle.TleError):
        tle.PagedChunkBatch(c.cache, c.tables, [1000, 0], [1, 1])
    with pytest.raises(ValueError):
        tle.PagedKVCache(8, 64, c.cache.shape, pools=(plain.key_pool, plain.value_pool[:, :4]))
    with pytest.raises(ValueError):
        tle.PagedKVCache(8, 64, c.cache.shape, dtype=bf, pools=(plain.key_pool, plain.value_pool))
    given = tle.PagedKVCache(8, 64, c.cache.shape, pools=(plain.key_pool, plain.value_pool))
    assert given.key_pool.data_ptr() == plain.key_pool.data_ptr()


def test_buffers_outlive_work_on_another_stream(cuda):
    """A batch that is dropped while its call waits on a stream of its own:
    what the allocator hands out next does not reach that call."""
    import torch
    import tle
    c = Case([3000, 40], [60, 2], seed=16)
    want = torch.zeros_like(c.out)
    c.batch.attend(c.q, want, c.layer)
    side = torch.cuda.Stream()
    gate = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):
            gate = gate @ gate * 1e-2          # keeps the stream busy
        c.batch.attend(c.q, c.out, c.layer)
    sizes = [(t.numel(), t.dtype) for t in (c.batch._desc_dev, c.batch.workspace)]
    c.batch = None
    for n, dt in sizes * 4:
        torch.full((n,), 77, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    assert torch.equal(c.out, want) and tle.device_error() == 0


def test_set_positions_replans(cuda):
    """The same batch object over growing contexts and other chunk lengths."""
    c = Case([900, 60, 3000], [300, 200, 400], seed=10)
    for pos, new in (([0, 0, 0], [5, 1, 0]), ([5, 1, 0], [1, 1, 1]), ([6, 2, 1], [200, 0, 300]), ([900, 60, 3000], [300, 200, 400])):
        c.pos, c.new, c.T = pos, new, sum(new)
        c.batch.set_positions(pos, new)
        check_attend(c)


def test_two_batches_in_flight(cuda):
    """Two batches (own workspaces) over one cache on two streams at once."""
    import torch
    import tle
    a = Case([2500, 100], [30, 1], seed=11)
    other = tle.PagedChunkBatch(a.cache, a.tables, a.pos, a.new)
    a.batch.attend(a.q, a.out, a.layer)
    torch.cuda.synchronize()
    want = a.out.clone()
    outs = [torch.zeros_like(a.out) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, s, o in zip((a.batch, other), streams, outs):
            b.attend(a.q, o, a.layer, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_bad_page_ids_are_reported_not_read(cuda, act):
    """An id outside the pool: its rows count as zeros and 0x105 is recorded;
    append stores nothing there."""
    import torch
    import tle
    c = Case([130], [6], act=act, seed=12)
    good = c.tables[0].clone()
    for bad in (c.cache.n_pages, -1, 1 << 30):
        c.tables[0].copy_(good)
        c.tables[0][1] = bad
        c.batch.attend(c.q, c.out, c.layer)
        torch.cuda.synchronize()
        assert tle.device_error() == 0x105
        c.tables[0].copy_(good)
        kp, vp = c.cache.key_pool.clone(), c.cache.value_pool.clone()
        page = int(good[1])
        c.cache.key_pool[c.layer, page] = 0
        c.cache.value_pool[c.layer, page] = 0
        got = c.out.clone()
        check_attend(c)
        assert torch.equal(got, c.out)
        c.cache.key_pool.copy_(kp)
        c.cache.value_pool.copy_(vp)
    c.tables[0][2] = c.cache.n_pages          # rows 128 .. 191 hold the six new ones
    before = (c.cache.key_pool.clone(), c.cache.value_pool.clone())
    c.batch.append(None, c.k, c.v, c.layer)
    torch.cuda.synchronize()
    assert tle.device_error() == 0x105
    assert torch.equal(before[0], c.cache.key_pool) and torch.equal(before[1], c.cache.value_pool)


def test_offsets_past_32_bits(cuda):
    """Pages whose rows lie more than 2^32 bytes and 2^31 elements into the pools."""
    import torch
    import tle
    page, n_pages = 65536, 140                                   # 9.2 M rows, 4.7 GB a pool
    shape = tle.Shape(1, 32, 4, HD, BASE)
    dims = (1, n_pages, page, 256)
    kp, vp = (torch.empty(dims, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = tle.PagedKVCache(n_pages, page, shape, dtype=torch.bfloat16, pools=(kp, vp))
    c = Case([10], [3], seed=13, layers=1)
    c.cache, c.page = cache, page
    c.pos, c.new, c.T = [300, 70], [5, 1], 6
    c.tables = [torch.tensor([139], dtype=torch.int32, device="cuda"), torch.tensor([131], dtype=torch.int32, device="cuda")]
    g = torch.Generator(device="cuda").manual_seed(13)
    for t in c.tables:
        for pool in (kp, vp):
            pool[0, int(t[0]), :400] = torch.randn(400, 256, generator=g, device="cuda").to(torch.bfloat16)
    c.q = torch.randn(6, 2048, generator=g, device="cuda")
    c.k, c.v = (torch.randn(6, 256, generator=g, device="cuda") for _ in range(2))
    c.out = torch.zeros_like(c.q)
    c.batch = tle.PagedChunkBatch(cache, c.tables, c.pos, c.new)
    c.batch.append(None, c.k, c.v, 0)
    want, size = rotated(c.k, c.positions())
    rows = np.concatenate([c.flat_rows(s, np.arange(p, p + m)) for s, (p, m) in enumerate(zip(c.pos, c.new))])
    got = kp[0].view(-1, 256)[torch.from_numpy(rows).cuda()].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -8 + size * 2.0 ** -21)
    check_attend(c)


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("act,pool", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("kw", [
    dict(pos=[0], new=[1]), dict(pos=[63, 0, 200], new=[2, 0, 65]), dict(pos=[3000, 17], new=[33, 1], page=256),
    dict(pos=[40], new=[9], heads=(7, 1)), dict(pos=[70, 131], new=[45, 130], heads=(20, 4)),
    dict(pos=[5], new=[3], heads=(8, 8)), dict(pos=[100000], new=[2], page=1024)])
def test_append_matches_the_formula(cuda, act, pool, kw):
    import torch
    import tle
    c = Case(**kw, act=act, pool=pool, seed=20, pad=2)
    p = c.positions()
    before = (c.cache.key_pool.clone(), c.cache.value_pool.clone())
    q0, k0 = c.q.clone(), c.k.clone()
    c.batch.append(c.q, c.k, c.v, c.layer, q_out=c.out)
    torch.cuda.synchronize()
    assert torch.equal(q0, c.q) and torch.equal(k0, c.k)
    want, size = rotated(c.q[:c.T], p)
    got = c.out[:c.T].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= np.abs(want) * U[act] + size * 2.0 ** -21)
    assert bool((c.out[c.T:] == 7.0).all())
    rows = np.concatenate([c.flat_rows(s, np.arange(a, a + m)) for s, (a, m) in enumerate(zip(c.pos, c.new))])
    at = torch.from_numpy(rows).cuda()
    want, size = rotated(c.k[:c.T], p)
    got = c.cache.key_pool[c.layer].view(-1, c.KH * HD)[at].double().cpu().numpy()
    assert np.all(np.abs(got - want) <= np.abs(want) * U[pool] + size * 2.0 ** -21)
    got = c.cache.value_pool[c.layer].view(-1, c.KH * HD)[at]
    assert torch.equal(got, c.v[:c.T].to(got.dtype))
    for new, old in zip((c.cache.key_pool, c.cache.value_pool), before):   # nothing else is written
        old[c.layer].view(-1, c.KH * HD)[at] = new[c.layer].view(-1, c.KH * HD)[at]
        assert torch.equal(new, old)
    assert tle.device_error() == 0


def test_append_in_place_strided_and_unrotated(cuda):
    import torch
    c = Case([90, 300], [33, 2], seed=21)
    qkv = torch.randn(c.T, 40 * HD, device="cuda")
    q, k, v = qkv[:, :32 * HD], qkv[:, 32 * HD:36 * HD], qkv[:, 36 * HD:]
    c.batch.append(q, k, v, c.layer, q_out=c.out)
    a = (c.out.clone(), c.cache.key_pool.clone(), c.cache.value_pool.clone())
    qq = q.contiguous()
    c.batch.append(qq, k.contiguous(), v.contiguous(), c.layer, q_out=qq)      # q in place
    torch.cuda.synchronize()
    assert torch.equal(qq, a[0]) and torch.equal(c.cache.key_pool, a[1]) and torch.equal(c.cache.value_pool, a[2])
    c.batch.append(q, k, v, c.layer, rotate=False, q_out=c.out)
    torch.cuda.synchronize()
    assert torch.equal(c.out, q)
    rows = np.concatenate([c.flat_rows(s, np.arange(p, p + m)) for s, (p, m) in enumerate(zip(c.pos, c.new))])
    assert torch.equal(c.cache.key_pool[c.layer].view(-1, 256)[torch.from_numpy(rows).cuda()], k.to(torch.bfloat16))


# ---------------------------------------------------------- used together
def test_pieces_of_a_prompt_equal_the_whole_and_decode_goes_on(cuda):
    """A prompt appended and attended in pieces gives the rows and results of
    the whole prompt at once; the framework's paged decode of the next token
    agrees with a chunk of one (bf16 precision, its contract)."""
    import torch
    import tle
    n = 333
    whole = Case([0], [n], page=64, seed=30)
    whole.batch.run(whole.q, whole.k, whole.v, whole.out, 1)
    parts = Case([0], [n], page=64, seed=30)
    at = 0
    for m in (1, 63, 64, 100, 1, 104):
        b = tle.PagedChunkBatch(parts.cache, parts.tables, [at], [m])
        s = slice(at, at + m)
        b.run(parts.q[s], parts.k[s], parts.v[s], parts.out[s], 1)
        at += m
    torch.cuda.synchronize()
    assert torch.equal(whole.cache.key_pool, parts.cache.key_pool)
    assert torch.equal(whole.cache.value_pool, parts.cache.value_pool)
    turned = torch.empty_like(whole.q)
    whole.batch.append(whole.q, whole.k, whole.v, 1, q_out=turned)
    want, tol = attention64(whole, turned)
    for c in (whole, parts):
        assert bool(((c.out.double() - want).abs() <= tol).all())
    # the next token: framework decode, then the chunk of one on the same cache
    pos = n - 1                                  # decode the last token again
    dec = tle.PagedDecodeBatchBf16(whole.cache, [whole.tables[0]], [pos])
    one = tle.PagedChunkBatch(whole.cache, [whole.tables[0]], [pos], [1])
    q, k, v = whole.q[pos:], whole.k[pos:], whole.v[pos:]
    a, b = torch.zeros(1, 2048, device="cuda"), torch.zeros(1, 2048, device="cuda")
    dec.run(q, k, v, a, 1)
    rows = whole.cache.key_pool.clone()
    one.run(q, k, v, b, 1)
    torch.cuda.synchronize()
    assert float((a - b).abs().max()) <= 2e-2
    near = (rows.float() - whole.cache.key_pool.float()).abs() <= rows.float().abs() * 2.0 ** -7 + 1e-30
    assert bool(near.all())
    assert tle.device_error() == 0


def test_prompt_into_an_fp32_cache_then_the_framework_decode(cuda):
    """append into fp32 pools holds what the paged fp32 decode expects: its
    result over those rows is the formula's (decode contract, 1e-4)."""
    import torch
    import tle
    c = Case([0, 0], [130, 40], page=16, pool="f32", seed=31)
    c.batch.append(c.q, c.k, c.v, c.layer, q_out=c.out)
    dec = tle.PagedDecodeBatch(c.cache, c.tables, [129, 39])
    last = torch.tensor([129, 169], device="cuda")
    out = torch.zeros(2, 2048, device="cuda")
    dec.run(c.q[last], c.k[last], c.v[last], out, c.layer)
    torch.cuda.synchronize()
    want, _ = attention64(c, c.out)
    assert float((out.double() - want[last]).abs().max()) <= 1e-4


def test_a_serving_step_with_sampling(cuda):
    """Prompt pieces, one decode step, logits under rules, a token: each
    stage through its public call, the token the 64-bit formula's."""
    import torch
    import tle
    V = 1000
    c = Case([0, 64, 500], [70, 1, 3], act="bf16", seed=32)
    c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    last = torch.tensor([69, 70, 73], device="cuda")
    W = torch.randn(2048, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) / 45
    logits = c.out[last].float() @ W
    hist = torch.tensor([5, 5, 9, 11, 5], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 3, 3, 5], dtype=torch.int32, device="cuda")
    allowed = torch.full((3, -(-V // 32)), -1, dtype=torch.int32, device="cuda")
    top = int(logits[1].argmax())
    allowed[1, top // 32] &= ~(1 << (top % 32)) if top % 32 < 31 else 0x7FFFFFFF
    f = lambda *x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    rules = tle.LogitRules(3, V, tokens=hist, token_start=start, repetition=f(1.5, 2, 1.1), frequency=f(.5, .1, .2),
                           presence=f(.2, .3, .1), allowed=allowed)
    adj = torch.empty_like(logits)
    tle.logits_adjust(adj, logits, rules)
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    for r in range(3):
        tle.sample_argmax(adj[r], tok[r:r + 1])
    torch.cuda.synchronize()
    assert torch.equal(tok.long(), adj.argmax(1)) and int(tok[1]) != top
    assert tle.device_error() == 0


# ------------------------------------------- captured calls and larger plans
def grown(c, pos, new, room):
    """c's batch over tables for `room` rows per sequence, planned for pos, new."""
    import torch
    import tle
    c.page = 64
    c.cache = tle.PagedKVCache(len(pos) * (room // 64) + 1, 64, c.cache.shape, dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(77)
    for pool in (c.cache.key_pool, c.cache.value_pool):
        pool.copy_(torch.randn(pool.shape, generator=g, device="cuda"))
    c.tables = [c.cache.table(c.cache.alloc(room // 64)) for _ in pos]
    c.batch = tle.PagedChunkBatch(c.cache, c.tables, pos, new)


@pytest.mark.parametrize("pos,new,large", [
    ([700], [1], ([5000], [1])),                        # the same tokens, more pieces: a larger workspace
    ([700], [1], ([6000], [300])),                      # more tokens: descriptor and q buffer too
    ([700, 3], [5, 40], ([4000, 5000], [60, 200])),
])
def test_a_replay_after_a_larger_plan_uses_no_freed_buffer(cuda, pos, new, large):
    """Captured under a small plan, replayed after a larger one replaced the
    batch's buffers: 0x10b and nothing is written, neither pools nor results
    nor memory that was handed out since; right again under the small plan."""
    import torch
    import tle
    c = Case(pos, new, seed=40)
    grown(c, pos, new, 6400)
    c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    graph.replay()
    torch.cuda.synchronize()
    want, plan = c.out.clone(), bytes(c.batch.plan)
    held = [t for t in (c.batch._desc_dev, c.batch.workspace, c.batch._q[c.q.dtype])]
    places = [(t.data_ptr(), t.numel() * t.element_size()) for t in held]
    sizes = [(t.numel(), t.dtype) for t in held]
    del held
    big = Case(large[0], large[1], seed=41)
    c.batch.set_positions(*large)
    assert bytes(c.batch.plan) != plan
    c.batch.run(big.q, big.k, big.v, big.out, c.layer)
    torch.cuda.synchronize()
    others = [torch.full((n * 4 if dt == torch.uint8 else n,), 77, dtype=dt, device="cuda") for n, dt in sizes for _ in range(8)]
    for t in others:                                    # what the graph uses is nobody else's
        a, n = t.data_ptr(), t.numel() * t.element_size()
        assert all(a + n <= p or p + m <= a for p, m in places)
    pools = (c.cache.key_pool.clone(), c.cache.value_pool.clone())
    c.out.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert tle.device_error() == 0x10b
    assert bool((c.out == 3).all())
    assert torch.equal(pools[0], c.cache.key_pool) and torch.equal(pools[1], c.cache.value_pool)
    c.batch.set_positions(pos, new)
    assert bytes(c.batch.plan) == plan
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c.out, want) and tle.device_error() == 0
    c.out.fill_(3)
    c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    torch.cuda.synchronize()
    assert torch.equal(c.out, want)
    assert all(bool((t == 77).all()) for t in others)


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_shorter_descriptor_of_another_plan_does_nothing(cuda, act):
    """Calls with a plan whose records would lie behind the end of the
    descriptor that they are given: 0x10b, nothing is written."""
    import ctypes
    import torch
    import tle
    c = Case([3000, 40, 20], [100, 1, 300], act=act, seed=42)
    small = tle.PagedChunkBatch(c.cache, c.tables[:1], [0], [1])
    n = small.plan.desc_bytes
    desc = small._desc_dev[:n].clone()
    assert n < c.batch.plan.desc_bytes / 10 and c.batch.plan.n_merge > 0
    pools = (c.cache.key_pool.clone(), c.cache.value_pool.clone())
    L, pool, plan, code = tle.lib(), c.cache.pool(), c.batch.plan, [tle.TLE_ACT_F32, tle.TLE_ACT_BF16][act == "bf16"]
    stream = torch.cuda.current_stream().cuda_stream
    c.out.fill_(3)
    rc = L.tle_append_bf16_paged(ctypes.byref(c.cache.shape), ctypes.addressof(pool), ctypes.byref(plan), desc.data_ptr(),
                                 c.q.data_ptr(), 2048, c.k.data_ptr(), 256, c.v.data_ptr(), 256, c.out.data_ptr(), code, 0, 1,
                                 stream)
    assert rc == tle.TLE_OK and tle.device_error() == 0x10b
    rc = L.tle_prefill_bf16_paged(ctypes.byref(c.cache.shape), ctypes.addressof(pool), ctypes.byref(plan), desc.data_ptr(),
                                  c.q.data_ptr(), 2048, c.out.data_ptr(), 2048, code, 0, c.batch.workspace.data_ptr(),
                                  c.batch.workspace.numel() * 4, stream)
    assert rc == tle.TLE_OK and tle.device_error() == 0x10b
    assert bool((c.out == 3).all())
    assert torch.equal(pools[0], c.cache.key_pool) and torch.equal(pools[1], c.cache.value_pool)


def test_run_on_a_stream_takes_memory_of_that_stream(cuda):
    """The buffer of the rotated q is not one that work still pending on
    another stream writes to."""
    import torch
    c = Case([900, 40], [200, 57], seed=43)
    want = torch.empty_like(c.out)
    c.batch.run(c.q, c.k, c.v, want, c.layer)
    torch.cuda.synchronize()
    c.batch._q.clear()
    del c.batch._old[:]
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    pending = torch.empty_like(c.q)
    at = pending.data_ptr()
    gate = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        gate = gate @ gate * 1e-2
    pending.fill_(77.0)
    del pending                                          # free for this stream, not for others
    c.batch.run(c.q, c.k, c.v, c.out, c.layer, stream=side)
    assert c.batch._q[c.q.dtype].data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(c.out, want)


def test_plans_are_not_made_in_a_capture(cuda):
    """set_positions uploads from a host buffer that it gives back: recorded in
    a graph, a replay would upload whatever is there then.  Refused."""
    import torch
    import tle
    c = Case([100, 20], [3, 4], seed=44)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            c.batch.set_positions([101, 21], [3, 4])
        with pytest.raises(RuntimeError):
            tle.PagedChunkBatch(c.cache, c.tables, [100, 20], [3, 4])
        c.batch.attend(c.q, c.out, c.layer)
    graph.replay()
    torch.cuda.synchronize()
    want, tol = attention64(c, c.q)
    assert bool(((c.out.double() - want).abs() <= tol).all())
    assert tle.device_error() == 0


# ------------------------------------------------- infinities in attended rows
def infinite_keys(c, rows):
    """Scores of -inf at these rows of sequence 0 for every head: an infinity in
    one column of K against q of one sign there."""
    c.q.view(c.q.shape[0], c.H, HD)[:, :, 5] = c.q.view(c.q.shape[0], c.H, HD)[:, :, 5].abs() + 0.1
    import torch
    at = torch.from_numpy(c.flat_rows(0, np.array(rows, np.int64))).cuda()
    c.cache.key_pool[c.layer].view(-1, c.KH, HD)[at, :, 5] = -float("inf")


def attention64_without(c, rows):
    """attention64 of c (one sequence), the rows' weights 0; NaN where a token
    attends to nothing else."""
    import torch
    p, m, G = c.pos[0], c.new[0], c.H // c.KH
    out = torch.zeros(m, c.H * HD, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    at = torch.from_numpy(c.flat_rows(0, np.arange(p + m))).cuda()
    hide = torch.arange(p + m, device="cuda")[None, :] > p + torch.arange(m, device="cuda")[:, None]
    gone = torch.zeros(p + m, dtype=torch.bool, device="cuda")
    gone[torch.tensor(rows, device="cuda")] = True
    hide = hide | gone
    for h in range(c.H):
        sl = slice((h // G) * HD, (h // G + 1) * HD)
        k = c.cache.key_pool[c.layer].view(-1, c.KH * HD)[at, sl].double()
        v = c.cache.value_pool[c.layer].view(-1, c.KH * HD)[at, sl].double()
        k[gone] = 0
        qq = c.q[:m, h * HD:(h + 1) * HD].double()
        e = qq @ k.T / 8
        big = (qq.abs() @ k.abs().T / 8).masked_fill(hide, 0).amax(1, keepdim=True)
        top = e.abs().masked_fill(hide, 0).amax(1, keepdim=True)
        w = torch.softmax(e.masked_fill(hide, -float("inf")), 1)
        vv = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
        o, size = w @ vv, w @ vv.abs()
        rel = 2 * (big * 2.0 ** -17 + top * 2.0 ** -23 + 2.0 ** -22) + ((p + m) / 16 + 16) * 2.0 ** -23
        if c.act == "bf16":
            rel = rel + 2.0 ** -8 + 2.0 ** -12
        out[:, h * HD:(h + 1) * HD] = o
        tol[:, h * HD:(h + 1) * HD] = rel * size + U[c.act] * (o.abs() + rel * size)
    return out, tol


def check_keys_of_no_weight(c, keys, bad=None):
    import torch
    import tle
    infinite_keys(c, keys)
    sees = torch.zeros(c.T, dtype=torch.bool, device="cuda")
    if bad is not None:
        row = int(c.flat_rows(0, np.array([bad]))[0])
        c.cache.value_pool[c.layer].view(-1, c.KH * HD)[row] = float("nan")
        sees = torch.arange(c.T, device="cuda") + c.pos[0] >= bad
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    want, tol = attention64_without(c, keys)
    some = torch.isfinite(want).all(1) & ~sees
    assert bool(some.any()) and bool(((c.out.double() - want).abs() <= tol)[some].all())
    assert bool((~torch.isfinite(c.out[sees])).all())
    assert tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,keys,bad", [([200], [3], [0], 201), ([1000], [20], list(range(140)), 1019),
                                              ([130], [2], list(range(128)), 131)])
def test_keys_of_no_weight_beside_a_bad_row(cuda, act, pos, new, keys, bad):
    """Rows whose score is -inf come first, a NaN in V behind some tokens of the
    same block: the tokens that do not attend to it have the formula's finite
    results."""
    check_keys_of_no_weight(Case(pos, new, act=act, seed=50, max_ctas=1), keys, bad)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,keys,bad", [
    ([200], [3], [0], None), ([200], [1], [0, 150], None), ([3000], [2], [1, 700, 2999], None),       # few rows
    ([0], [70], [1], 40), ([100], [300], [0, 1, 2, 50], 260), ([5000], [20], [17, 4000], None),       # many, in pieces
    ([1000], [40], list(range(140)), None), ([130], [16], list(range(128)), None)])
@pytest.mark.parametrize("values", ["full", "halves"])
def test_keys_of_no_weight(cuda, act, pos, new, keys, bad, values):
    """An infinity in K whose scores are -inf takes its row out and leaves the
    results finite, for q of 24 bits and for q that a bf16 number holds (whose
    lower terms are zero)."""
    import torch
    c = Case(pos, new, act=act, seed=51)
    if values == "halves":
        c.q = c.q.to(torch.bfloat16).to(c.q.dtype)
        c.q[:, 5::64] = 0.4                              # + 0.1: 0.5 in the column with the infinity
    check_keys_of_no_weight(c, keys, bad)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([900], [70]), ([900], [2])])
def test_keys_of_no_weight_in_place(cuda, act, pos, new):
    """The same with out = q: rows computed again read their q first."""
    import torch
    c = Case(pos, new, act=act, seed=52)
    infinite_keys(c, [3, 400])
    c.batch.attend(c.q, c.out, c.layer)
    c.batch.attend(c.q, c.q, c.layer)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(c.out).all()) and torch.equal(c.q, c.out)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,max_ctas", [([0], [1], 0), ([0], [40], 1), ([90], [3], 1), ([300], [20], 1), ([300], [60], 1),
                                              ([900], [3], 0), ([5000], [20], 0), ([5000], [70], 0)])
def test_rows_without_any_weight(cuda, act, pos, new, max_ctas):
    """Scores of -inf only: 0/0, whether the plan cuts the item or not; the
    tokens that see one other row have that row of V."""
    import torch
    import tle
    c = Case(pos, new, act=act, seed=53, max_ctas=max_ctas)
    last = pos[0] + new[0] - 1
    infinite_keys(c, list(range(last)))
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    assert bool(torch.isnan(c.out[:-1]).all())
    if last:
        v = c.cache.value_pool[c.layer].view(-1, c.KH, HD)[int(c.flat_rows(0, np.array([last]))[0])]
        got = c.out[-1].view(c.KH, -1, HD).double()
        assert bool(((got - v[:, None].double()).abs() <= 2.0 ** -21 * v[:, None].abs()).all())
    infinite_keys(c, [last])
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    assert bool(torch.isnan(c.out).all()) and tle.device_error() == 0


@pytest.mark.parametrize("pool", ["f32", "bf16"])
def test_calls_follow_the_cache_to_other_memory(cuda, pool):
    """Pools whose storage was exchanged under the same tensor objects: the
    next call reads and writes the new one."""
    import torch
    import tle
    c = Case([90, 30], [20, 3], pool=pool, seed=54)
    other = Case([90, 30], [20, 3], pool=pool, seed=55)      # tables of the same sizes
    c.batch.append(c.q, c.k, c.v, c.layer, q_out=c.out)
    torch.cuda.synchronize()
    old = (c.cache.key_pool.detach(), c.cache.value_pool.detach())   # the storage itself
    before = tuple(t.clone() for t in old)
    c.cache.key_pool.data, c.cache.value_pool.data = (t.clone() for t in (other.cache.key_pool, other.cache.value_pool))
    c.batch.append(c.q * 2, c.k * 2, c.v * 2, c.layer, q_out=c.out)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(old, before))
    rows = np.concatenate([c.flat_rows(s, np.arange(p, p + m)) for s, (p, m) in enumerate(zip(c.pos, c.new))])
    got = c.cache.value_pool[c.layer].view(-1, 256)[torch.from_numpy(rows).cuda()]
    assert torch.equal(got, (c.v * 2).to(got.dtype))
    if pool == "bf16":
        check_attend(c)
    assert tle.device_error() == 0


def test_what_a_batch_keeps_is_bounded(cuda):
    """Batches that grow by a token at a time: all the buffers ever kept are at
    most three times the newest ones."""
    import torch
    c = Case([0, 900], [200, 200], page=64, seed=56, layers=1)
    for n in range(20, 200):
        c.batch.set_positions([0, 5 * n], [n, 1])
        c.batch.run(c.q, c.k, c.v, c.out, 0)
    torch.cuda.synchronize()
    b = c.batch
    size = lambda ts: sum(t.numel() * t.element_size() for t in ts)  # noqa: E731
    newest = size([b._desc_dev, b.workspace, *b._q.values()])
    assert size([*b._descs, b.workspace, *b._q.values(), *b._old]) <= 3 * newest
    assert b._q[c.q.dtype].shape[0] < 2 * 200
    b.set_positions(c.pos, c.new)
    check_attend(c)
