"""Appends by rules, 8-bit pages and their attention (tle_append_rules_*,
tle_append_q8_paged, tle_read_q8_paged, tle_prefill_q8_paged) against the
formulas in 64 bits.

Tolerances, per value (u = half a step of a type, relative: bf16 2^-8, fp32
2^-24):
* a norm: a sum of 64 squares in 32 bits (at most 64 roundings of 2^-24), a mean, a root, a
  quotient and two products: 2^-17 relative, all in all;
* a rotation: sine and cosine are off by 2 ulp (2^-23), times the factor (a
  rounding), two products and a sum: (|a| + |b|) factor 2^-21, plus u of the stored type;
* a stored 8-bit value: half a step of its row's scale from the number that was
  stored, which is off as above; the scale is the formula's unless the largest
  element is that near to the border;
* attend: as for bf16 pages (a score is off by 2^-17 sum|q k| / 8 at most, a
  weight by 2 (that + |s| 2^-23 + 2^-22) relative, the sum over rows by (rows / 16 +
  16) 2^-23; with bf16 activations and many rows a weight is rounded to bf16).
  Weights of few rows are fp16 pairs whose smallest step is 2^-24 where the largest
  weight times V's power of two is 2^7 at least: rows * 2^-32 of the largest
  such product, times 128.
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
    return {"f32": torch.float32, "bf16": torch.bfloat16, "q8": torch.int8}[name]


def power(e):
    """2^e of whole numbers, exactly."""
    import torch
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def to8(x):
    """Codes and scale bytes of rows x [..., 64] of finite numbers, by the definition in 64 bits."""
    import torch
    most = x.double().abs().amax(-1)
    e = torch.ceil(torch.log2(most.clamp(min=2.0 ** -140) / 127)).clamp(min=-126)
    e = torch.where(127 * power(e) < most, e + 1, e)
    e = torch.where((127 * power(e - 1) >= most) & (e > -126), e - 1, e)
    e = e.clamp(max=121)                                   # of larger numbers the values would not be finite
    codes = torch.round(x.double() / power(e)[..., None]).clamp(-127, 127)
    return codes.to(torch.int8), (e + 127).to(torch.uint8)


def from8(codes, scale):
    import torch
    f = power(scale.long() - 127)
    f = torch.where(scale == 255, torch.full_like(f, float("inf")), f)
    return codes.double() * f[..., None]


class Case:
    """A paged cache of random rows and a batch over it, on the GPU."""

    def __init__(self, pos, new, heads=(32, 4), page=64, act="f32", pool="q8", layers=2, seed=0, spare=3, pad=0,
                 max_ctas=0, scale=1.0, sizes=False):
        import torch
        import tle
        self.pos, self.new, self.page, self.act, self.pool = list(pos), list(new), page, act, pool
        self.H, self.KH = heads
        self.layers, self.layer = layers, layers - 1
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-(p + m) // page) for p, m in zip(pos, new)]
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        self.tables, at = [], 0
        for k in need:
            self.tables.append(ids[at:at + k].clone())
            at += k
        self.cache = c = tle.PagedKVCache(n_pages, page, tle.Shape(layers, self.H, self.KH, HD, BASE), dtype=dtype(pool))
        rnd = lambda *d: torch.randn(d, generator=g, device="cuda")  # noqa: E731
        if pool == "q8":
            for codes, sc in ((c.key_pool, c.key_scale), (c.value_pool, c.value_scale)):
                x = rnd(*codes.shape)
                if sizes and codes is c.value_pool:         # rows of very different sizes
                    x *= torch.exp2(torch.randint(-18, 19, x.shape[:-1], generator=g, device="cuda").float())[..., None]
                a, b = to8(x)
                codes.copy_(a)
                sc.copy_(b)
        else:
            c.key_pool.copy_(rnd(*c.key_pool.shape))
            c.value_pool.copy_(rnd(*c.value_pool.shape))
        T = self.T = sum(new)
        self.q, self.k, self.v = rnd(T + pad, self.H * HD).to(dtype(act)) * scale, *(rnd(T + pad, self.KH * HD).to(dtype(act)) for _ in range(2))
        self.out = torch.full_like(self.q, 7.0)
        self.batch = tle.PagedChunkBatch(c, self.tables, pos, new, max_ctas=max_ctas)

    def positions(self):
        return np.concatenate([np.arange(p, p + m) for p, m in zip(self.pos, self.new)] or [[]]).astype(np.int64)

    def places(self, s, rows):
        """(page ids, rows in the page) of rows of sequence s, as index tensors."""
        import torch
        t = self.tables[s].cpu().numpy().astype(np.int64)
        return torch.from_numpy(t[rows // self.page]).cuda(), torch.from_numpy(rows % self.page).cuda()

    def new_places(self):
        import torch
        got = [self.places(s, np.arange(p, p + m)) for s, (p, m) in enumerate(zip(self.pos, self.new))]
        return torch.cat([a for a, _ in got]), torch.cat([b for _, b in got])

    def stored(self, what, page, row):
        """Values of rows of the layer, 64-bit [rows][kv_heads][64]."""
        c, l = self.cache, self.layer
        pool, sc = (c.key_pool, c.key_scale) if what == "k" else (c.value_pool, c.value_scale)
        if self.pool != "q8":
            return pool[l][page, row].double().view(-1, self.KH, HD)
        return from8(pool[l][page, :, row], sc[l][page, :, row])


def headed(c, x, layout, R, freq, factor, norm, eps, rotate=True):
    """64-bit norm and rotation of x [T][heads * 64]: results and tolerances."""
    import torch
    y = x[:c.T].double().view(c.T, -1, HD)
    rel = 0.0
    if norm is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * norm.double()
        rel = 2.0 ** -17
    tol = rel * y.abs()
    if rotate:
        a = (c.positions().astype(np.float32)[:, None] * np.asarray(freq, np.float32)).astype(np.float64)
        cos, sin = (torch.from_numpy(f(a)).cuda()[:, None] * factor for f in (np.cos, np.sin))
        i, j = (torch.arange(R // 2), torch.arange(R // 2, R)) if layout == "half" else (torch.arange(0, R, 2), torch.arange(1, R, 2))
        p, q = y[..., i], y[..., j]
        size = (p.abs() + q.abs()) * (rel + 2.0 ** -21) * max(factor, 1.0)
        y, tol = y.clone(), tol.clone()
        y[..., i], y[..., j] = p * cos - q * sin, p * sin + q * cos
        tol[..., i] = tol[..., j] = size
    return y, tol


APPENDS = [
    dict(pos=[0], new=[1]), dict(pos=[5, 63, 64, 200], new=[1, 1, 3, 0]),
    dict(pos=[0, 100], new=[130, 7], page=128, heads=(16, 8)),
    dict(pos=[4000], new=[9], heads=(7, 1), page=1024), dict(pos=[60, 1], new=[5, 300], heads=(12, 4)),
    dict(pos=[i * 7 for i in range(70)], new=[1] * 70, heads=(8, 8)),
]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pool", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("i", range(len(APPENDS)))
@pytest.mark.parametrize("layout,R,scaling,norms", [
    ("half", 64, "none", "qk"), ("interleaved", 64, "yarn", ""), ("half", 32, "linear", "q"), ("interleaved", 48, "ntk", "k"),
    ("half", 16, "none", "qk"), ("half", 48, "yarn", ""), ("interleaved", 16, "none", "q")])
def test_append_by_rules(cuda, act, pool, i, layout, R, scaling, norms):
    import torch
    import tle
    c = Case(**APPENDS[i], act=act, pool=pool, seed=i, pad=2)
    freq, factor = tle.rope_frequencies(R, BASE, scaling, 4.0, 2048)
    w = {x: 1 + 0.3 * torch.randn(HD, generator=c.g, device="cuda") for x in norms}
    rules = tle.AppendRules(layout, inv_freq=freq, rope_factor=factor, q_norm=w.get("q"), k_norm=w.get("k"), eps=1e-5)
    before = [t.clone() for t in (c.cache.key_pool, c.cache.value_pool)]
    c.batch.append(c.q, c.k, c.v, c.layer, q_out=c.out, rules=rules)
    torch.cuda.synchronize()
    assert tle.device_error() == 0
    q, tq = headed(c, c.q, layout, R, freq, factor, w.get("q"), 1e-5)
    k, tk = headed(c, c.k, layout, R, freq, factor, w.get("k"), 1e-5)
    v = c.v[:c.T].double().view(c.T, -1, HD)
    got = c.out[:c.T].double().view(c.T, -1, HD)
    assert bool(((got - q).abs() <= tq + U[act] * (q.abs() + tq)).all())
    assert bool((c.out[c.T:] == 7).all())                 # rows behind the last token
    page, row = c.new_places()
    for what, x, t, exact in (("k", k, tk, False), ("v", v, torch.zeros_like(v), True)):
        y = c.stored(what, page, row)
        if pool != "q8":
            assert bool(((y - x).abs() <= t + U[pool] * (x.abs() + t)).all())
            continue
        P, S = (c.cache.key_pool, c.cache.key_scale) if what == "k" else (c.cache.value_pool, c.cache.value_scale)
        codes, sc = P[c.layer][page, :, row], S[c.layer][page, :, row]
        if exact:
            want, ws = to8(x)
            assert torch.equal(codes, want) and torch.equal(sc, ws)
            continue
        most, far = x.abs().amax(-1), t.amax(-1)
        step = power(sc.long() - 127)
        assert bool((most - far <= 127 * step).all()) and bool(((most + far > 63.5 * step) | (sc == 1)).all())
        assert bool(((y - x).abs() <= step[..., None] / 2 + t).all()) and int(codes.abs().max()) <= 127
    # nothing else was written
    for t, b in zip((c.cache.key_pool, c.cache.value_pool), before):
        mine = torch.zeros(t.shape[:2] + (c.page,), dtype=torch.bool, device="cuda")
        mine[c.layer, page, row] = True
        mine = mine[:, :, None, :, None].expand_as(t) if pool == "q8" else mine[..., None].expand_as(t)
        assert torch.equal(t[~mine], b[~mine])


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_append_into_8_bits_without_rules_is_the_frameworks_rope(cuda, act):
    """q and k as tle_append_paged rotates them; norms without rotation; keys and values only; strided and in place."""
    import torch
    import tle
    c, d = Case([10, 700], [3, 40], act=act), Case([10, 700], [3, 40], act=act, pool="f32")
    c.batch.append(c.q, c.k, c.v, 1, q_out=c.out)
    d.batch.append(c.q, c.k, c.v, 1, q_out=d.out)
    page, row = c.new_places()
    rotated = d.stored("k", *d.new_places())
    pair = lambda x: x.double().view(x.shape[0], -1, HD // 2, 2).abs().sum(-1).repeat_interleave(2, -1) * 2.0 ** -21  # noqa: E731
    u = U[act] * d.out.double().abs() * 2
    assert bool(((c.out.double() - d.out.double()).abs() <= pair(c.q).view(c.q.shape) + u).all())
    step = power(c.cache.key_scale[1][page, :, row].long() - 127)[..., None]
    assert bool(((c.stored("k", page, row) - rotated).abs() <= step / 2 + pair(c.k)).all())
    want = c.cache.key_pool[1][page, :, row]
    keep = [t.clone() for t in (c.cache.key_pool, c.cache.value_pool, c.cache.key_scale, c.cache.value_scale)]
    wide = torch.zeros(c.T, (c.H + 2 * c.KH) * HD + 8, dtype=c.q.dtype, device="cuda")
    wide[:, :c.H * HD], wide[:, c.H * HD:(c.H + c.KH) * HD], wide[:, (c.H + c.KH) * HD:-8] = c.q, c.k, c.v
    q, k, v = wide[:, :c.H * HD], wide[:, c.H * HD:(c.H + c.KH) * HD], wide[:, (c.H + c.KH) * HD:-8]
    c.cache.key_pool.zero_()
    c.cache.value_scale.zero_()
    out2 = torch.empty_like(c.out)
    c.batch.append(q, k, v, 1, q_out=out2)
    assert torch.equal(out2, c.out) and torch.equal(c.cache.key_pool[1][page, :, row], want)
    c.cache.key_pool.copy_(keep[0]), c.cache.value_scale.copy_(keep[3])
    mine = c.q.clone()
    c.batch.append(mine, c.k, c.v, 1, q_out=mine)
    assert torch.equal(mine, c.out)
    c.batch.append(None, c.k, c.v, 1)
    for t, b in zip((c.cache.key_pool, c.cache.value_pool, c.cache.key_scale, c.cache.value_scale), keep):
        assert torch.equal(t, b)
    w = torch.rand(HD, device="cuda") + 0.5
    c.batch.append(c.q, c.k, c.v, 1, rotate=False, q_out=out2, rules=tle.AppendRules("half", q_norm=w, eps=0.25))
    x, t = headed(c, c.q, "half", 64, [], 1.0, w, 0.25, rotate=False)
    assert bool(((out2.double().view(x.shape) - x).abs() <= t + U[act] * x.abs() * 1.01).all())
    want, ws = to8(c.k.double().view(c.T, -1, HD))
    assert torch.equal(c.cache.key_pool[1][page, :, row], want) and torch.equal(c.cache.key_scale[1][page, :, row], ws)
    assert tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_rows_at_the_ends_of_the_range(cuda, act):
    """Zeros, the smallest and largest numbers, a border of the scale, infinities and NaN; read back."""
    import torch
    import tle
    c = Case([3], [12], act=act, heads=(4, 4))
    v = c.v
    big = float(torch.finfo(v.dtype).max)
    tiny = 2.0 ** -133 if act == "bf16" else 2.0 ** -149
    v[0] = 0
    v[1], v[2] = tiny, -tiny
    v[3] = big
    v[4] = torch.where(torch.arange(256, device="cuda") % 2 == 0, big, -big)
    v[5] = 127.0
    v[6] = 127.0
    v[6, ::64] = 127.5 if act == "bf16" else float(np.nextafter(np.float32(127), np.float32(128)))
    v[7] = 2.0 ** -126
    v[8, 7], v[8, 64 + 3], v[8, 128 + 63] = float("inf"), -float("inf"), float("nan")
    v[9] = torch.arange(256, device="cuda") % 64 * 2.0 - 63.0      # ties: odd halves of a step of 2
    v[9, ::64] = 254.0
    v[10] = 2.0 ** -120 * torch.randn(256, device="cuda")
    c.batch.append(None, c.k, v, 1, rotate=False)
    page, row = c.new_places()
    fine = torch.isfinite(v.double().view(-1, c.KH, HD)).all(-1)
    want, ws = to8(torch.where(fine[..., None], v.double().view(-1, c.KH, HD), 0))
    codes, sc = c.cache.value_pool[1][page, :, row], c.cache.value_scale[1][page, :, row]
    assert torch.equal(codes[fine], want[fine]) and torch.equal(sc[fine], ws[fine])
    assert bool((sc[~fine] == 255).all()) and bool((codes[~fine] == 0).all()) and int((~fine).sum()) == 3
    for t in ("f32", "bf16"):
        k_out, v_out = (torch.full((12, 256), 3.0, dtype=dtype(t), device="cuda") for _ in range(2))
        c.batch.read(k_out, v_out, 1, new_only=True)
        got = v_out.double().view(-1, c.KH, HD)
        assert torch.equal(got[fine], from8(codes, sc)[fine]) and bool(torch.isnan(got[~fine]).all())
    assert tle.device_error() == 0


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(pos=[0], new=[1]), dict(pos=[5, 63, 64, 200, 9], new=[1, 1, 3, 0, 120]), dict(pos=[1000, 3], new=[40, 257], page=128, heads=(8, 1)),
    dict(pos=[(37 * i) % 300 for i in range(600)], new=[i % 3 for i in range(600)], heads=(4, 2)),   # more sequences than threads
    dict(pos=[20000, 9, 15000], new=[1, 1, 1], page=1024)])
def test_read_gives_the_stored_values(cuda, t, kw):
    import torch
    import tle
    c = Case(**kw, seed=9, layers=3)
    c.layer = 1
    order = [(s, p + m) for s, (p, m) in enumerate(zip(c.pos, c.new)) if m]
    at = [c.places(s, np.arange(n)) for s, n in order]
    page, row = torch.cat([a for a, _ in at]), torch.cat([b for _, b in at])
    n = c.batch.n_rows
    assert n == page.numel()
    w = c.KH * HD
    k_out = torch.full((n + 2, w + 16), 5.0, dtype=dtype(t), device="cuda")
    v_out = torch.full((n + 2, w), 5.0, dtype=dtype(t), device="cuda")
    c.batch.read(k_out[:, 8:8 + w], v_out, 1)
    torch.cuda.synchronize()
    for got, what in ((k_out[:n, 8:8 + w], "k"), (v_out[:n], "v")):
        assert torch.equal(got.double().reshape(n, c.KH, HD), c.stored(what, page, row))
    assert bool((k_out[:, :8] == 5).all()) and bool((k_out[:, 8 + w:] == 5).all())
    assert bool((k_out[n:] == 5).all()) and bool((v_out[n:] == 5).all())
    one = torch.zeros(n, w, dtype=dtype(t), device="cuda")
    c.batch.read(None, one, 1)
    assert torch.equal(one, v_out[:n])
    fresh = torch.zeros(c.T, w, dtype=dtype(t), device="cuda")
    c.batch.read(fresh, None, 1, new_only=True)
    assert torch.equal(fresh.double().view(-1, c.KH, HD), c.stored("k", *c.new_places()))
    assert tle.device_error() == 0


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
        page, row = c.places(s, np.arange(p + m))
        K, V = c.stored("k", page, row), c.stored("v", page, row)
        top_v = power(c.cache.value_scale[c.layer][page, :, row].long() - 127) * 128
        for h in range(c.H):
            k, v = K[:, h // G], V[:, h // G]
            qq = q[t0:t0 + m, h * HD:(h + 1) * HD].double()
            e = qq @ k.T / 8
            hide = torch.arange(p + m, device="cuda")[None, :] > p + torch.arange(m, device="cuda")[:, None]
            big = (qq.abs() @ k.abs().T / 8).masked_fill(hide, 0).amax(1, keepdim=True)
            top = e.abs().masked_fill(hide, 0).amax(1, keepdim=True)
            w = torch.softmax(e.masked_fill(hide, -float("inf")), 1)
            o, size = w @ v, w @ v.abs()
            rel = 2 * (big * 2.0 ** -17 + top * 2.0 ** -23 + 2.0 ** -22) + ((p + m) / 16 + 16) * 2.0 ** -23
            if c.act == "bf16" and m * G > 32:
                rel = rel + 2.0 ** -8 + 2.0 ** -12
            least = (p + m) * 2.0 ** -32 * (w * top_v[:, h // G]).amax(1, keepdim=True)
            out[t0:t0 + m, h * HD:(h + 1) * HD] = o
            tol[t0:t0 + m, h * HD:(h + 1) * HD] = rel * size + least + U[c.act] * (o.abs() + rel * size)
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
    assert tle.device_error() == 0
    assert bool((d <= tol).all()), float((d / tol).max())


ATTENDS = [
    dict(pos=[0], new=[1]), dict(pos=[0], new=[4]), dict(pos=[0], new=[5]),
    dict(pos=[126, 127, 128, 129], new=[1, 1, 1, 1]),                   # around a tile's edge
    dict(pos=[14, 15, 16, 17, 63, 64], new=[1, 1, 1, 1, 1, 1]),         # around a step's and a copy's
    dict(pos=[63, 64, 0, 500], new=[1, 2, 3, 0]),                       # a sequence without tokens
    dict(pos=[300], new=[2]), dict(pos=[300], new=[3]),                 # 16 and 24 rows
    dict(pos=[1000, 3, 250], new=[40, 257, 1], page=128),               # many rows and few in one batch
    dict(pos=[2000, 1029, 1500, 2040], new=[1, 1, 1, 1], page=1024),
    dict(pos=[5000], new=[3]),                                          # one sequence over many CTAs
    dict(pos=[5000, 700], new=[9, 1]),
    dict(pos=[70, 131], new=[45, 30], heads=(8, 8)),                    # one query head per KV head
    dict(pos=[70, 131], new=[4, 130], heads=(12, 4)), dict(pos=[70, 131], new=[2, 3], heads=(20, 4), page=256),
    dict(pos=[70, 900], new=[1, 2], heads=(7, 1)), dict(pos=[90], new=[1], heads=(32, 1)),
    dict(pos=[64], new=[3], heads=(128, 1)),
    dict(pos=list(range(0, 1600, 25)), new=[1 + i % 5 for i in range(64)]),
    dict(pos=[900, 10, 400, 77], new=[100, 200, 300, 1], max_ctas=3),   # several items per CTA
    dict(pos=[900, 10, 400, 1300], new=[3, 2, 1, 4], max_ctas=1),
    dict(pos=[40] * 300, new=[1] * 300, heads=(4, 1), max_ctas=2),      # more pieces than a CTA holds records of
]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(ATTENDS)))
def test_attend_matches_the_formula(cuda, i, act):
    check_attend(Case(**ATTENDS[i], act=act, seed=i))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([700, 130], [1, 3]), ([700], [20])])
def test_attend_large_scores(cuda, act, pos, new):
    """Weights concentrated on a few rows (scores up to about +-100)."""
    check_attend(Case(pos, new, act=act, scale=25.0, seed=3))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([700, 130, 3000], [1, 3, 1])])
def test_attend_values_of_very_different_sizes(cuda, act, pos, new):
    """V rows from 2^-18 to 2^18: the largest contributions keep their precision whatever
    their softmax weights are."""
    check_attend(Case(pos, new, act=act, seed=4, sizes=True))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 9])
def test_attend_falling_and_rising_scores(cuda, act, new):
    """Scores that grow along the rows (every tile moves the running maxima) and that fall."""
    import torch
    for sign in (1.0, -1.0):
        c = Case([900], [new], act=act, seed=4)
        n = 900 + new
        ramp = torch.linspace(-1, 1, n, device="cuda") * sign * 6
        page, row = c.places(0, np.arange(n))
        codes, sc = to8(ramp[:, None, None].expand(n, c.KH, HD))
        c.cache.key_pool[c.layer][page, :, row] = codes
        c.cache.key_scale[c.layer][page, :, row] = sc
        c.q.abs_().mul_(3)
        check_attend(c)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([200], [3]), ([0, 60], [70, 1]), ([120], [150]), ([0], [1])])
def test_rows_nobody_attends_to_do_not_matter(cuda, act, pos, new):
    """Any bytes behind a sequence's last row, in other pages, other layers: the same bits."""
    import torch
    c = Case(pos, new, act=act, seed=5)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    keep = torch.zeros(c.cache.n_pages, c.page, dtype=torch.bool, device="cuda")
    for s, (p, m) in enumerate(zip(pos, new)):
        keep[c.places(s, np.arange(p + m))] = True
    away = ~keep[:, None].expand(-1, c.KH, -1)
    for codes, sc in ((c.cache.key_pool, c.cache.key_scale), (c.cache.value_pool, c.cache.value_scale)):
        codes[c.layer][away] = -128
        sc[c.layer][away] = 255
        codes[:c.layer], sc[:c.layer] = 127, 254
    check_attend(c)
    assert torch.equal(first, c.out)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new,at", [([200], [3], 201), ([0], [70], 40), ([100], [300], 260), ([5], [1], 2), ([1000], [4], 1003),
                                        ([1000], [1], 1000), ([130], [33], 3), ([3000], [2], 17)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_row_of_nan_reaches_only_the_tokens_that_attend_to_it(cuda, act, pos, new, at, where):
    import torch
    import tle
    c = Case(pos, new, act=act, seed=6)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    want, tol = attention64(c, c.q)
    page, row = c.places(0, np.array([at]))
    codes, sc = (c.cache.key_pool, c.cache.key_scale) if where == "k" else (c.cache.value_pool, c.cache.value_scale)
    codes[c.layer][page, 1, row], sc[c.layer][page, 1, row] = 0, 255    # KV head 1: query heads 8 .. 15
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    sees = torch.arange(new[0], device="cuda") + pos[0] >= at
    mine = slice(8 * HD, 16 * HD)
    assert bool(((c.out.double() - want).abs() <= tol)[~sees].all())
    assert torch.equal(c.out[:, :8 * HD], first[:, :8 * HD]) and torch.equal(c.out[:, 16 * HD:], first[:, 16 * HD:])
    assert bool(torch.isnan(c.out[sees, mine]).all()) and tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_a_bad_q_reaches_only_its_head(cuda, act, bad):
    import torch
    c = Case([200, 70], [2, 1], act=act, seed=7)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    c.q[1, 3 * HD + 5] = float(bad)
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    hit = torch.zeros_like(c.out, dtype=torch.bool)
    hit[1, 3 * HD:4 * HD] = True
    assert bool(torch.isnan(c.out[hit]).all()) and torch.equal(c.out[~hit], first[~hit])


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** 40])
def test_q_and_k_of_extreme_sizes(cuda, act, size):
    import torch
    c = Case([300, 40], [1, 3], act=act, seed=8)
    c.q.mul_(size)
    c.cache.key_scale.copy_(c.cache.key_scale.int() - int(np.log2(size)))
    check_attend(c)
    c.q.zero_()
    check_attend(c)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([100, 900], [2, 3]), ([100, 900], [20, 3])])
def test_attend_strides_in_place_and_rows_behind(cuda, act, pos, new):
    import torch
    c = Case(pos, new, act=act, seed=10, pad=3)
    check_attend(c)
    assert bool((c.out[c.T:] == 7).all())
    want = c.out.clone()
    wide = torch.full((c.T + 3, c.H * HD + 24), 3.0, dtype=c.q.dtype, device="cuda")
    wide[:, 8:8 + c.H * HD] = c.q
    out = torch.full((c.T + 3, c.H * HD + 8), 3.0, dtype=c.q.dtype, device="cuda")
    c.batch.attend(wide[:, 8:8 + c.H * HD], out[:, :c.H * HD], c.layer)
    assert torch.equal(out[:c.T, :c.H * HD], want[:c.T]) and bool((out[:, c.H * HD:] == 3).all()) and bool((out[c.T:] == 3).all())
    c.batch.attend(c.q, c.q, c.layer)
    assert torch.equal(c.q[:c.T], want[:c.T])


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("pos,new", [([300, 5000], [1, 2]), ([300, 900, 64], [40, 3, 0])])
def test_attend_is_reproducible_replays_and_follows_a_plan_of_the_same_numbers(cuda, act, pos, new):
    import torch
    import tle
    c = Case(pos, new, act=act, seed=11)
    c.batch.attend(c.q, c.out, c.layer)
    first = c.out.clone()
    for _ in range(3):
        c.batch.attend(c.q, c.out, c.layer)
        assert torch.equal(c.out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.batch.attend(c.q, c.out, c.layer)
        c.batch.attend(c.out, c.out, c.layer)              # the workspace used twice in one graph
    c.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    again = torch.empty_like(c.out)
    c.batch.attend(first, again, c.layer)
    assert torch.equal(again, c.out) and tle.device_error() == 0
    c.batch.set_positions([p // 2 for p in pos], [m - 1 if m else 0 for m in new])   # another plan
    c.out.fill_(5.0)
    graph.replay()
    torch.cuda.synchronize()
    assert tle.device_error() == 0x10b and bool((c.out == 5).all())
    c.batch.set_positions(pos, new)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, c.out) and tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_bad_page_ids_are_reported_not_read(cuda, act):
    """Ids outside the pool: their rows count as zeros, in the attention and in read; appends skip them."""
    import torch
    import tle
    for pos, new in (([200, 90], [1, 1]), ([200, 90], [40, 1])):
        c = Case(pos, new, act=act, seed=12)
        keep = c.tables[0].clone()
        page, row = c.places(0, np.arange(64, 128))
        c.tables[0][1] = 1 << 30
        c.batch.attend(c.q, c.out, c.layer)
        k_out = torch.full((c.batch.n_rows, 256), 3.1415, device="cuda")   # no value of 8 bits
        torch.cuda.synchronize()
        assert tle.device_error() == 0x105
        c.batch.read(k_out, None, c.layer)
        torch.cuda.synchronize()
        assert tle.device_error() == 0x105 and bool((k_out[64:128] == 0).all()) and bool(((k_out[:64] - 3.1415).abs() > 1e-6).all())
        c.tables[0].copy_(keep)
        for codes in (c.cache.key_pool, c.cache.value_pool):
            codes[c.layer][page, :, row] = 0
        want, tol = attention64(c, c.q)
        assert bool(((c.out.double() - want).abs() <= tol).all())
        before = [t.clone() for t in (c.cache.key_pool, c.cache.key_scale)]
        last = (pos[0] // 64)
        c.tables[0][last:] = -1
        c.batch.append(None, c.k, c.v, c.layer)
        c.batch.read(k_out[:c.T], None, c.layer, new_only=True)
        torch.cuda.synchronize()
        assert tle.device_error() == 0x105
        gone, r = c.places(1, np.arange(90, 91))
        for t, b in zip((c.cache.key_pool, c.cache.key_scale), before):
            t[c.layer][gone, :, r] = b[c.layer][gone, :, r]
            assert torch.equal(t, b)


def test_a_workspace_without_room_is_reported(cuda):
    """A replaced plan of the same numbers with more rows than the workspace has
    room for: 0x10c, no write outside it, the chunks of few rows right."""
    import ctypes
    import torch
    import tle
    c = Case([500, 900], [1, 40], seed=13)
    b = c.batch
    check_attend(c)
    want = c.out.clone()
    n = b._ws_bytes
    at = n - 3 * (2 * 128 * 256 * 2 + 4)                   # three staged pages too few
    room = torch.full((n + 4096,), 77, dtype=torch.uint8, device="cuda")
    pool = c.cache.pool()
    c.out.zero_()
    rc = tle.lib().tle_prefill_q8_paged(b._shape_ref, ctypes.addressof(pool), ctypes.byref(b.plan), b._desc_dev.data_ptr(), c.q.data_ptr(),
                                        2048, c.out.data_ptr(), 2048, 0, c.layer, room.data_ptr(), at, None)
    assert rc == 0
    torch.cuda.synchronize()
    assert tle.device_error() == 0x10c and bool((room[at:] == 77).all()) and torch.equal(c.out[:1], want[:1])
    with pytest.raises(tle.TleError):
        k_out = torch.zeros(4, 256, device="cuda")
        tle._check(tle.lib().tle_read_q8_paged(b._shape_ref, ctypes.addressof(pool), ctypes.byref(b.plan), b._desc_dev.data_ptr(),
                                               k_out.data_ptr(), 256, None, 0, 4, 0, c.layer, 1, None))
    k_out = torch.full((100, 256), 3.1415, device="cuda")  # fewer rows than there are
    assert tle.lib().tle_read_q8_paged(b._shape_ref, ctypes.addressof(pool), ctypes.byref(b.plan), b._desc_dev.data_ptr(), k_out.data_ptr(),
                                       256, None, 0, 90, 0, c.layer, 0, None) == 0
    torch.cuda.synchronize()
    assert tle.device_error() == 0x10c and bool((k_out[90:] == k_out[99, 0]).all()) and bool((k_out[:90] != k_out[99, 0]).all())


@pytest.mark.parametrize("new", [1, 4])
def test_long_fp32_sums_do_not_drift(cuda, new):
    """16000 rows of equal weights and V of one sign: the sum over rows is that of 32-bit numbers."""
    import torch
    c = Case([16000], [new], page=1024, seed=14, layers=1)
    c.q.mul_(1e-3)
    c.cache.value_pool.copy_(c.cache.value_pool.abs().clamp(min=1))
    c.batch.attend(c.q, c.out, 0)
    torch.cuda.synchronize()
    want, _ = attention64(c, c.q)
    assert float(((c.out.double() - want).abs() / want.abs()).max()) <= 2.0 ** -19


def test_offsets_past_32_bits(cuda):
    """Pools of more than 2^32 bytes: rows at their end are stored, read and attended to."""
    import torch
    import tle
    n_pages, page = 70000, 256                             # 4.6 GB of codes in each pool
    cache = tle.PagedKVCache(n_pages, page, tle.Shape(1, 32, 4, HD, BASE), dtype=torch.int8)
    cache.key_scale.fill_(120), cache.value_scale.fill_(120)
    table = torch.tensor([n_pages - 1, 0, n_pages - 2], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(600, w, device="cuda") for w in (2048, 256, 256))
    b = tle.PagedChunkBatch(cache, [table], [0], [600])
    b.append(None, k, v, 0, rotate=False)
    out = torch.zeros(600, 256, device="cuda")
    b.read(None, out, 0)
    a, s = to8(v.view(600, 4, HD))
    assert torch.equal(out.double().view(600, 4, HD), from8(a, s))
    b.set_positions([599], [1])
    got = torch.zeros(1, 2048, device="cuda")
    b.attend(q[:1], got, 0)
    torch.cuda.synchronize()
    a, s = to8(k.view(600, 4, HD))
    K, V = from8(a, s), out.double().view(600, 4, HD)
    w = torch.softmax(torch.einsum("hd,rhd->hr", q[0].double().view(32, HD), K.repeat_interleave(8, 1)) / 8, 1)
    want = torch.einsum("hr,rhd->hd", w, V.repeat_interleave(8, 1)).reshape(1, 2048)
    assert float((got - want).abs().max()) <= 1e-5 and tle.device_error() == 0


def test_other_streams_and_two_batches(cuda):
    """Two batches on two streams at once, each with its workspace."""
    import torch
    import tle
    cs = [Case([700, 40, 300], [1, 50, 4], seed=20 + i) for i in range(2)]
    for c in cs:
        c.batch.run(c.q, c.k, c.v, c.out, c.layer)
    torch.cuda.synchronize()
    want = [c.out.clone() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        for c, s in zip(cs, streams):
            c.out.zero_()
        torch.cuda.synchronize()
        for c, s in zip(cs, streams):
            c.batch.run(c.q, c.k, c.v, c.out, c.layer, stream=s)
        torch.cuda.synchronize()
        assert all(torch.equal(c.out, w) for c, w in zip(cs, want))
    assert tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_prompt_in_pieces_then_decode_steps(cuda, act):
    """A prompt stored and attended to in pieces, then single tokens, by rules with norms: each
    step against the formula over what the cache holds, and the stored rows independent of the pieces."""
    import torch
    import tle
    c = Case([0, 0], [150, 33], act=act, seed=30, layers=1)
    w = torch.rand(HD, device="cuda") + 0.5
    freq, factor = tle.rope_frequencies(32, scaling="yarn", factor=2.0)
    rules = tle.AppendRules("half", inv_freq=freq, rope_factor=factor, q_norm=w, k_norm=w)
    c.batch.append(None, c.k, c.v, 0, rules=rules)
    whole = [t.clone() for t in (c.cache.key_pool, c.cache.key_scale, c.cache.value_pool, c.cache.value_scale)]
    for t in (c.cache.key_pool, c.cache.key_scale, c.cache.value_pool, c.cache.value_scale):
        t.zero_()
    starts, done = np.array([0, 150]), [0, 0]
    q, k, v = c.q, c.k, c.v
    for step in ([100, 30], [46, 0], [3, 1], [1, 2]):
        rows = np.concatenate([np.arange(s + d, s + d + n) for s, d, n in zip(starts, done, step)])
        c.pos, c.new, c.T = list(done), step, sum(step)
        c.batch.set_positions(done, step)
        qs, ks, vs = (x[torch.from_numpy(rows).cuda()].contiguous() for x in (q, k, v))
        turned, out = torch.empty_like(qs), torch.empty_like(qs)
        c.batch.append(qs, ks, vs, 0, q_out=turned, rules=rules)
        c.batch.attend(turned, out, 0)
        want, tol = attention64(c, turned)
        assert bool(((out.double() - want).abs() <= tol).all())
        both = torch.empty_like(qs)
        c.batch.run(qs, ks, vs, both, 0, rules=rules)
        assert torch.equal(both, out)
        done = [d + n for d, n in zip(done, step)]
    for s, n in ((0, 150), (1, 33)):
        page, row = c.places(s, np.arange(n))
        for a, b in zip((c.cache.key_pool, c.cache.key_scale, c.cache.value_pool, c.cache.value_scale), whole):
            assert torch.equal(a[0][page, :, row], b[0][page, :, row])
    assert tle.device_error() == 0


def test_tensors_and_caches_are_checked(cuda):
    import torch
    import tle
    c = Case([10], [3])
    b, w = c.batch, c.KH * HD
    z = lambda *d, t=torch.float32, dev="cuda": torch.zeros(d, dtype=t, device=dev)  # noqa: E731
    for bad in (lambda: b.read(z(12, w), None, 1), lambda: b.read(z(13, w - 8), None, 1), lambda: b.read(z(13, w), z(13, w, t=torch.bfloat16), 1),
                lambda: b.read(z(13, w, dev="cpu"), None, 1), lambda: b.read(None, None, 1), lambda: b.read(z(2, w), None, 1, new_only=True),
                lambda: b.read(z(13, w, t=torch.float16), None, 1),
                lambda: tle.AppendRules("other"), lambda: tle.AppendRules(inv_freq=[1.0] * 5, rotary_dim=16),
                lambda: tle.AppendRules(q_norm=z(63)), lambda: tle.AppendRules(q_norm=z(64, t=torch.bfloat16)),
                lambda: tle.AppendRules(k_norm=z(64, dev="cpu")), lambda: tle.rope_frequencies(scaling="other"),
                lambda: tle.PagedKVCache(4, 64, dtype=torch.int8, pools=(z(22, 4, 4, 64, 64, t=torch.int8),) * 2),
                lambda: tle.PagedKVCache(4, 64, dtype=torch.int8, pools=(z(22, 4, 64, 256, t=torch.int8),) * 2 + (z(22, 4, 4, 64, t=torch.uint8),) * 2)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: b.append(c.q, c.k, c.v, 1, q_out=c.out, rules=tle.AppendRules(rotary_dim=24)),
                lambda: b.append(c.q, c.k, c.v, 1, q_out=c.out, rules=tle.AppendRules(eps=-1.0)),
                lambda: b.read(z(13, w + 4)[:, :w], None, 1), lambda: b.read(z(13, w), None, 2),
                lambda: tle.rope_frequencies(24), lambda: tle.rope_frequencies(scaling="linear", factor=0.5)):
        with pytest.raises(tle.TleError):
            bad()
    d = Case([10], [3], pool="bf16")
    with pytest.raises(ValueError):
        d.batch.read(z(13, w), None, 1)
    assert tle.device_error() == 0
