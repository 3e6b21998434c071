"""Sampling of rows (tle_sample_rows) against the definition in 64 bits.

The choice is by sums of weights: the kernel's are whole numbers of 2^-40 of the
largest weight, so a sum over V tokens is off by V 2^-41 at most, and a choice has to be the
oracle's wherever no border (the end of the nucleus, the drawn number) is
nearer than NEAR = 2 V 2^-41 + 2^-45 times the sum; there are few such rows.
"""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tinyllama-engine_b200"))

pytestmark = pytest.mark.gpu


def oracle(x, T, k, p, m, u):
    """(token, distance of the nearest border over the sum) of one row of float32 logits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1, 1.0
    if not T > 0:
        return int(order[0]), 1.0
    V, near = len(x), 1.0
    keep = order[:k] if 0 < k < V else order
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x[keep] - top) / float(T))
    w = np.where(x[keep] == top, 1.0, np.where(np.isnan(w), 0.0, w))
    if m > 0:
        near = min(near, float(np.min(np.abs(w[1:] / min(m, 1.0) - 1.0), initial=1.0))) if m < 1 else near
        w = w[w >= min(m, 1.0)]
    w = w[w > 0]
    if p < 1:
        sums = np.cumsum(w)
        n = 1 + int(np.searchsorted(sums, max(p, 0.0) * sums[-1]))
        near = min(near, float(np.min(np.abs(sums - max(p, 0.0) * sums[-1]))) / sums[-1]) if p > 0 else near
        w = w[:n]
    by = np.argsort(keep[:len(w)])
    sums = np.cumsum(w[by])
    t = min(max(u, 0.0), 1.0) * sums[-1]
    at = min(int(np.searchsorted(sums, t, side="right")), len(by) - 1)
    near = min(near, float(np.min(np.abs(sums[:-1] - t), initial=sums[-1])) / sums[-1])
    return int(keep[by[at]]), near


def dev(a):
    import torch
    return torch.from_numpy(np.array(a)).cuda()


def run(x, T=None, k=None, p=None, m=None, u=None, stream=None, xs=None):
    import torch
    import tle
    n, V = x.shape
    f = lambda a: None if a is None else dev(np.broadcast_to(np.asarray(a, np.float32), n))  # noqa: E731
    rules = tle.SampleRules(n, V, f(T), None if k is None else dev(np.broadcast_to(np.asarray(k, np.int32), n)), f(p), f(m))
    out = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    t = dev(x) if xs is None else xs
    before = t.clone()
    tle.sample_rows(out, t, rules, f(u), stream=stream)
    torch.cuda.synchronize()
    assert tle.device_error() == 0 and torch.equal(t.view(torch.int32) if t.is_contiguous() else t, before.view(torch.int32) if t.is_contiguous() else before)
    return out.cpu().numpy()


def check(x, T=1.0, k=0, p=1.0, m=0.0, u=0.5, most_near=0.1):
    n, V = x.shape
    T, k, p, m, u = (np.broadcast_to(np.asarray(a, d), n) for a, d in ((T, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32)))
    got = run(x, T, k, p, m, u)
    near = 0
    for r in range(n):
        want, border = oracle(x[r], float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]))
        if border <= 2 * V * 2.0 ** -41 + 2.0 ** -45:
            near += 1
            continue
        assert got[r] == want, (r, int(got[r]), want, float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]), border)
    assert near <= max(1, most_near * n)
    return got


SIZES = [(1, 1), (1, 2), (3, 5), (2, 31), (7, 512), (5, 513), (1, 1000), (4, 4097), (64, 1023), (1, 32000), (2, 32000), (70, 32000), (3, 100003),
         (1, 200001), (1, 262144), (20, 50257)]


@pytest.mark.parametrize("n,V", SIZES)
@pytest.mark.parametrize("rules", ["none", "k", "p", "m", "kp", "kpm"])
def test_matches_the_definition(cuda, n, V, rules):
    r = np.random.default_rng(n * 1000 + V)
    x = (3 * r.standard_normal((n, V))).astype(np.float32)
    x[r.random((n, V)) < 0.1] = -np.inf
    x[:, r.integers(0, V)] = 1.0
    T = r.uniform(0.3, 1.5, n)
    T[r.random(n) < 0.1] = 0
    check(x, T, np.minimum((V ** r.random(n)).astype(int), V) if "k" in rules else 0, r.uniform(0, 1, n) if "p" in rules else 1.0,
          10 ** r.uniform(-5, 0, n) if "m" in rules else 0.0, r.random(n))


@pytest.mark.parametrize("rules", ["none", "k", "p", "kp"])
def test_ties(cuda, rules):
    """Few different logits, whole rows of one, -0 and 0: ties count by index."""
    r = np.random.default_rng(5)
    x = r.integers(-3, 4, (40, 3001)).astype(np.float32)
    x[:4] = 2.5
    x[4:8] = np.where(r.random((4, 3001)) < 0.5, -0.0, 0.0)
    x[8:12] = np.where(r.random((4, 3001)) < 0.99, -50.0, 0.0)
    u = r.random(40)
    got = check(x, 1.0, r.integers(1, 3001, 40) if "k" in rules else 0, r.uniform(0.01, 0.999, 40) if "p" in rules else 1.0, 0.0, u)
    if rules == "none":
        assert np.array_equal(got[:8], (u[:8].astype(np.float32).astype(np.float64) * 3001).astype(int))


def test_the_number_walks_the_row(cuda):
    """Equal weights of a power of two of tokens: the token is floor(u n), at 0 and just below 1 too."""
    x = np.full((1, 4096), -np.inf, np.float32)
    places = np.arange(7, 4096, 8)                          # 512 of them
    x[:, places] = 3.0
    for j in (0, 1, 255, 256, 511):
        for u in (j / 512, float(np.nextafter(np.float32((j + 1) / 512), np.float32(0)))):
            assert run(x, 1.0, u=u)[0] == places[j]
    for u, j in ((-1.0, 0), (float("nan"), 0), (1.0, 511), (7.0, 511)):   # outside [0, 1)
        assert run(x, 1.0, u=u)[0] == places[j]


def test_rows_without_a_choice(cuda):
    inf, nan = np.inf, np.nan
    x = np.zeros((9, 600), np.float32)
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, 77] = -1e30                                        # one token allowed
    x[3] = nan
    x[3, 599] = -3e38
    x[4, 5] = inf                                           # +inf: certain
    x[5, [9, 300]] = inf                                    # two of them
    x[6, 3] = nan
    x[6, 4] = 1.0
    x[7] = -3.4e38
    x[7, 8] = 3.4e38                                        # a difference that overflows
    x[8] = 1e-42                                            # subnormal, equal
    for kw in ({}, dict(k=10), dict(p=0.9), dict(m=0.5), dict(k=300, p=0.5, m=0.1)):
        got = run(x, 0.7, u=0.75, **kw)
        assert got[0] == -1 and got[1] == -1 and got[2] == 77 and got[3] == 599 and got[4] == 5 and got[7] == 8
        assert got[5] == (300 if kw.get("p", 1) > 0.5 and kw.get("k", 10) >= 2 else 9), kw
        assert got[6] not in (3,)
    assert np.array_equal(run(x, 0.0, u=0.75)[[0, 1, 2, 3, 4, 5, 6, 7, 8]], [-1, -1, 77, 599, 5, 9, 4, 8, 0])
    assert np.array_equal(run(x, np.nan, u=0.75), run(x, -1.0, u=0.75))


@pytest.mark.parametrize("T", [1e-30, 1e-4, 0.05, 30.0, 1e6, 1e30, np.inf])
@pytest.mark.parametrize("rules", ["none", "kpm"])
def test_temperatures(cuda, T, rules):
    r = np.random.default_rng(11)
    x = (5 * r.standard_normal((12, 2500))).astype(np.float32)
    x[3] *= 1e-20
    x[4] *= 1e20
    x[5:8, ::2] = -np.inf                                   # masked tokens stay so at any temperature
    on = rules != "none"
    check(x, T, r.integers(2, 2500, 12) if on else 0, r.uniform(0.3, 1, 12) if on else 1.0, r.uniform(0, 0.01, 12) if on else 0.0, r.random(12))


@pytest.mark.parametrize("k,p,m", [(1, 1.0, 0.0), (0, 0.0, 0.0), (0, 1.0, 1.0), (0, 1.0, 5.0), (0, 1e-30, 0.0), (1, 0.5, 0.9), (0, -1.0, 0.0)])
def test_filters_that_leave_the_first(cuda, k, p, m):
    r = np.random.default_rng(12)
    x = r.standard_normal((30, 5000)).astype(np.float32)
    x[1] = 4.0
    want = x.argmax(1)
    got = run(x, 1.0, k, p, m, r.random(30))
    same = np.ones(30, bool)
    same[1] = not (m >= 1 and k == 0)                       # all of them are the largest
    assert np.array_equal(got[same], want[same])


def test_filters_that_are_off(cuda):
    r = np.random.default_rng(13)
    x = r.standard_normal((30, 5000)).astype(np.float32)
    u = r.random(30)
    want = run(x, None, u=u)
    for kw in (dict(k=0), dict(k=-5), dict(k=5000), dict(k=1 << 30), dict(p=1.0), dict(p=2.0), dict(p=np.nan), dict(m=0.0), dict(m=-1.0),
               dict(m=np.nan), dict(T=1.0), dict(T=1.0, k=0, p=1.0, m=0.0)):
        assert np.array_equal(run(x, kw.pop("T", None), u=u, **kw), want), kw


def test_shares_of_the_draws(cuda):
    """One row drawn with 20000 numbers evenly spaced: each token as often as its probability says."""
    r = np.random.default_rng(14)
    one = (2 * r.standard_normal(300)).astype(np.float32)
    n = 20000
    got = run(np.broadcast_to(one, (n, 300)).copy(), 0.8, u=(np.arange(n) + 0.5) / n)
    w = np.exp((one.astype(np.float64) - one.max()) / np.float64(np.float32(0.8)))
    assert np.abs(np.bincount(got, minlength=300) - n * w / w.sum()).max() <= 1.01
    assert np.all(np.diff(got) >= 0)


def test_the_choice_does_not_depend_on_the_batch(cuda):
    """A row alone and among others (another number of CTAs a row): the same token."""
    r = np.random.default_rng(15)
    x = (3 * r.standard_normal((200, 32000))).astype(np.float32)
    u, k, p = r.random(200), r.integers(0, 500, 200), r.uniform(0.5, 1.1, 200)
    all_ = run(x, 0.9, k, p, 0.001, u)
    for a, b in ((0, 1), (5, 30), (100, 190)):
        assert np.array_equal(run(x[a:b], 0.9, k[a:b], p[a:b], 0.001, u[a:b]), all_[a:b])


def test_strides_streams_and_replays(cuda):
    import torch
    import tle
    r = np.random.default_rng(16)
    x = (3 * r.standard_normal((9, 1001))).astype(np.float32)
    u, p = r.random(9), r.uniform(0.5, 1, 9)
    want = run(x, 0.9, 40, p, 0.0, u)
    for pad, at in ((7, 0), (16, 1), (3, 3)):
        wide = torch.full((9, 1001 + pad), 50.0, device="cuda")
        wide[:, at:at + 1001] = dev(x)
        view = wide[:, at:at + 1001]
        assert np.array_equal(run(x, 0.9, 40, p, 0.0, u, xs=view), want)
    side = torch.cuda.Stream()
    t = dev(x)
    torch.cuda.synchronize()
    assert np.array_equal(run(x, 0.9, 40, p, 0.0, u, stream=side, xs=t), want)
    rules = tle.SampleRules(9, 1001, dev(np.full(9, 0.9, np.float32)), dev(np.full(9, 40, np.int32)), dev(p.astype(np.float32)))
    out, uu = torch.zeros(9, dtype=torch.int32, device="cuda"), dev(u.astype(np.float32))
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        tle.sample_rows(out, t, rules, uu)
    for k in range(3):
        u2 = r.random(9)
        uu.copy_(dev(u2.astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), run(x, 0.9, 40, p, 0.0, u2))


def test_the_most_rows(cuda):
    import torch
    import tle
    n, V = 65535, 33
    x = torch.randn(n, V, device="cuda")
    out = torch.zeros(n, dtype=torch.int32, device="cuda")
    tle.sample_rows(out, x, tle.SampleRules(n, V, torch.zeros(n, device="cuda")), torch.zeros(n, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(out.long(), x.argmax(1))


def test_after_the_logit_rules(cuda):
    """A batch's last step: penalties and a mask, then a token for each row, as one chain."""
    import torch
    import tle
    r = np.random.default_rng(17)
    n, V = 6, 32000
    x = (3 * r.standard_normal((n, V))).astype(np.float32)
    words = r.integers(0, 1 << 32, (n, V // 32), dtype=np.uint64).astype(np.uint32)
    words[2] = 0                                             # allows nothing
    words[3] = 0
    words[3, 10] = 1 << 7                                    # one token
    adjusted = torch.empty(n, V, device="cuda")
    tle.logits_adjust(adjusted, dev(x), tle.LogitRules(n, V, allowed=dev(words.view(np.int32))))
    out = torch.zeros(n, dtype=torch.int32, device="cuda")
    u = r.random(n).astype(np.float32)
    rules = tle.SampleRules(n, V, dev(np.full(n, 0.8, np.float32)), dev(np.full(n, 50, np.int32)), dev(np.full(n, 0.9, np.float32)))
    tle.sample_rows(out, adjusted, rules, dev(u))
    torch.cuda.synchronize()
    bits = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")
    y = np.where(bits > 0, x, -np.inf).astype(np.float32)
    got = out.cpu().numpy()
    assert got[2] == -1 and got[3] == 10 * 32 + 7
    for i in range(n):
        want, near = oracle(y[i], float(np.float32(0.8)), 50, float(np.float32(0.9)), 0.0, float(u[i]))
        assert got[i] == want or near < 1e-6


def test_rules_and_tensors_are_checked(cuda):
    import torch
    import tle
    z = lambda *d, t=torch.float32, dev="cuda": torch.zeros(d, dtype=t, device=dev)  # noqa: E731
    i32 = torch.int32
    ok = tle.SampleRules(2, 100, z(2))
    for bad in (lambda: tle.SampleRules(2, 100, z(3)), lambda: tle.SampleRules(2, 100, z(2, t=torch.float64)), lambda: tle.SampleRules(2, 100, top_k=z(2)),
                lambda: tle.SampleRules(2, 100, top_p=z(2, dev="cpu")), lambda: tle.SampleRules(2, 100, min_p=z(4)[::2]),
                lambda: tle.sample_rows(z(2), z(2, 100), ok, z(2)), lambda: tle.sample_rows(z(3, t=i32), z(2, 100), ok, z(2)),
                lambda: tle.sample_rows(z(2, t=i32), z(2, 99), ok, z(2)), lambda: tle.sample_rows(z(2, t=i32), z(2, 200)[:, ::2], ok, z(2)),
                lambda: tle.sample_rows(z(2, t=i32), z(2, 100, t=torch.bfloat16), ok, z(2)), lambda: tle.sample_rows(z(2, t=i32), z(2, 100), ok, z(1)),
                lambda: tle.sample_rows(z(2, t=i32), z(2, 100, dev="cpu"), ok, z(2)), lambda: tle.sample_rows(z(2, t=i32, dev="cpu"), z(2, 100), ok, z(2))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(tle.TleError):
        tle.sample_rows(z(1, t=i32), z(1, 262145), tle.SampleRules(1, 262145), z(1))
    assert tle.device_error() == 0
