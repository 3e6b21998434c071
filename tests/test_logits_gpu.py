"""Logit rules (tle_logits_adjust) against the formulas in 64 bits.

A logit goes through at most: a quotient or product (one rounding, 2^-24 of
it), frequency * count and two differences (a rounding each), the sum of its
biases (one per entry) and its addition, so with m = |x| (rep or 1/rep) +
freq * count + pres + sum |bias| the result is within (5 + entries) 2^-24 m.
"""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tinyllama-engine_b200"))

pytestmark = pytest.mark.gpu


def dev(a, d=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if d is None else t.to(d)).cuda()


def make(n, V, hist, seed, pen=True, biases=0, mask=False, dup=False):
    """Host arrays of a case: logits and rules."""
    r = np.random.default_rng(seed)
    c = {"x": (3 * r.standard_normal((n, V))).astype(np.float32), "n": n, "V": V}
    if pen:
        counts = r.integers(0, hist + 1, n)
        c["token_start"] = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        c["tokens"] = r.integers(0, max(1, V // 8) if dup else V, int(counts.sum())).astype(np.int32)
        c["n_prompt"] = r.integers(0, hist // 2 + 1, n).astype(np.int32)
        c["repetition"] = r.uniform(0.8, 2, n).astype(np.float32)
        c["frequency"] = r.uniform(-0.5, 1, n).astype(np.float32)
        c["presence"] = r.uniform(-0.5, 1, n).astype(np.float32)
    if biases:
        k = r.integers(0, biases + 1, n)
        c["bias_start"] = np.concatenate([[0], np.cumsum(k)]).astype(np.int32)
        c["bias_tokens"] = r.integers(0, 5 if dup else V, int(k.sum())).astype(np.int32) % V
        c["bias_values"] = (5 * r.standard_normal(int(k.sum()))).astype(np.float32)
    if mask:
        c["allowed"] = r.integers(0, 1 << 32, (n, -(-V // 32)), dtype=np.uint64).astype(np.uint32).view(np.int32)
    return c


KEYS = ("tokens", "token_start", "n_prompt", "repetition", "frequency", "presence", "bias_tokens", "bias_values",
        "bias_start", "allowed")


def rules(c):
    import tle
    return tle.LogitRules(c["n"], c["V"], **{k: dev(c[k]) for k in KEYS if k in c})


def formula(c):
    """64-bit results, tolerances."""
    x = c["x"].astype(np.float64)
    size, terms = np.abs(x), np.zeros(x.shape)
    V = c["V"]
    for r in range(c["n"]):
        if "tokens" in c:
            ids = c["tokens"][c["token_start"][r]:c["token_start"][r + 1]]
            ids_ok = (ids >= 0) & (ids < V)
            made = ids[c["n_prompt"][r]:] if "n_prompt" in c else ids
            made = made[(made >= 0) & (made < V)]
            used = np.unique(ids[ids_ok])
            if "repetition" in c:
                rep = float(c["repetition"][r])
                x[r, used] = np.where(x[r, used] > 0, x[r, used] / rep, x[r, used] * rep)
                size[r, used] = np.maximum(size[r, used], np.abs(x[r, used]))
            times = np.bincount(made, minlength=V)
            f = float(c["frequency"][r]) if "frequency" in c else 0.0
            p = float(c["presence"][r]) if "presence" in c else 0.0
            x[r] -= f * times + p * (times > 0)
            size[r] += abs(f) * times + abs(p) * (times > 0)
        if "bias_tokens" in c:
            s = slice(c["bias_start"][r], c["bias_start"][r + 1])
            ids, b = c["bias_tokens"][s], c["bias_values"][s].astype(np.float64)
            fine = (ids >= 0) & (ids < V)
            np.add.at(x[r], ids[fine], b[fine])
            np.add.at(size[r], ids[fine], np.abs(b[fine]))
            np.add.at(terms[r], ids[fine], 1)
        if "allowed" in c:
            bits = np.unpackbits(c["allowed"][r].view(np.uint8), bitorder="little")[:V]
            x[r, bits == 0] = -np.inf
    return x, (5 + terms) * 2.0 ** -24 * size


def check(c, out):
    import torch
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want, tol = formula(c)
    inf = np.isneginf(want)
    assert np.array_equal(inf, np.isneginf(got))
    assert np.all(np.abs(got[~inf] - want[~inf]) <= tol[~inf])


@pytest.mark.parametrize("n,V,hist", [(1, 1, 3), (1, 31, 0), (3, 33, 50), (2, 4095, 100), (2, 4097, 300),
                                      (5, 32000, 700), (1, 100003, 4000), (70, 1001, 20)])
@pytest.mark.parametrize("pen,biases,mask", [(1, 0, 0), (0, 40, 0), (0, 0, 1), (1, 300, 1), (1, 5, 0), (0, 0, 0)])
def test_matches_the_formula(cuda, n, V, hist, pen, biases, mask):
    import torch
    import tle
    c = make(n, V, hist, seed=n * V + hist, pen=pen, biases=biases, mask=mask)
    x = dev(c["x"])
    out = torch.full_like(x, 7.0)
    tle.logits_adjust(out, x, rules(c))
    check(c, out)
    assert torch.equal(x, dev(c["x"]))
    tle.logits_adjust(x, x, rules(c))                  # in place
    torch.cuda.synchronize()
    assert torch.equal(x, out)
    assert tle.device_error() == 0


def test_tokens_listed_many_times(cuda):
    """Counts of many thousand; a token's biases are added in the list's
    order, the same bits in every call."""
    import torch
    import tle
    c = make(3, 500, 20000, seed=1, biases=2000, dup=True)
    c["bias_values"] *= np.float32(10) ** np.random.default_rng(2).integers(-4, 5, c["bias_values"].size).astype(np.float32)
    out = torch.empty(3, 500, device="cuda")
    R = rules(c)
    tle.logits_adjust(out, dev(c["x"]), R)
    check(c, out)
    for r in range(3):                                   # in order: the sums of 32-bit additions one by one
        s = slice(c["bias_start"][r], c["bias_start"][r + 1])
        acc = np.zeros(500, np.float32)
        for t, b in zip(c["bias_tokens"][s], c["bias_values"][s]):
            acc[t] = np.float32(acc[t] + b)
        only = {k: c[k] for k in ("n", "V", "bias_tokens", "bias_values", "bias_start")}
        z = torch.empty(3, 500, device="cuda")
        tle.logits_adjust(z, torch.zeros(3, 500, device="cuda"), rules(only))
        assert np.array_equal(z[r].cpu().numpy(), acc)
    again = torch.empty_like(out)
    tle.logits_adjust(again, dev(c["x"]), R)
    assert torch.equal(out, again)


@pytest.mark.parametrize("left_out", ["repetition", "frequency", "presence", "n_prompt"])
def test_single_penalties_left_out(cuda, left_out):
    import torch
    import tle
    c = make(4, 700, 90, seed=5)
    del c[left_out]
    if left_out == "n_prompt":
        pass                                             # every token counts as made
    out = torch.empty(4, 700, device="cuda")
    tle.logits_adjust(out, dev(c["x"]), rules(c))
    check(c, out)


def test_non_finite_logits_and_a_row_that_allows_nothing(cuda):
    import torch
    import tle
    c = make(3, 100, 0, seed=6, mask=True)
    c["tokens"] = np.arange(0, 60, 2).astype(np.int32)
    c["token_start"] = np.array([0, 30, 30, 30], np.int32)
    c["n_prompt"][:] = 0
    c["allowed"][1] = 0
    c["allowed"][0] = -1
    x = dev(c["x"])
    x[:, 0:10] = float("nan")
    x[:, 10:20] = float("inf")
    x[:, 20:30] = -float("inf")
    out = torch.empty_like(x)
    tle.logits_adjust(out, x, rules(c))
    torch.cuda.synchronize()
    assert bool(torch.isnan(out[0, :10]).all()) and bool((out[0, 10:20] == float("inf")).all())
    assert bool((out[0, 20:30] == -float("inf")).all())
    assert bool((out[1] == -float("inf")).all())         # even where a logit is NaN
    bits = torch.from_numpy(np.unpackbits(c["allowed"][2].view(np.uint8), bitorder="little")[:100]).cuda()
    assert bool((out[2][bits == 0] == -float("inf")).all())


@pytest.mark.parametrize("biases", [3, 200])
def test_a_bias_does_not_lift_the_mask(cuda, biases):
    """-inf where the mask says so, under an infinite or NaN bias too."""
    import torch
    import tle
    V = 90
    ids = np.arange(biases, dtype=np.int32) % V
    b = np.resize(np.array([np.inf, np.nan, -np.inf], np.float32), biases)
    words = np.full((1, 3), 0b1000, np.int32)          # every 32nd token from 3 on
    R = tle.LogitRules(1, V, bias_tokens=dev(ids), bias_values=dev(b), bias_start=dev(np.array([0, biases], np.int32)),
                       allowed=dev(words))
    out = torch.zeros(1, V, device="cuda")
    tle.logits_adjust(out, torch.ones(1, V, device="cuda"), R)
    ok = torch.arange(V, device="cuda") % 32 == 3
    assert bool((out[0][~ok] == -float("inf")).all())
    assert not bool((out[0][ok] == -float("inf")).all())


def test_the_most_rows(cuda):
    """65535 rows, each with a token list of its own."""
    import torch
    import tle
    n, V = 65535, 37
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(n, V, generator=g, device="cuda")
    ids = torch.randint(0, V, (n, 2), generator=g, device="cuda", dtype=torch.int32)
    rep = 1 + torch.rand(n, generator=g, device="cuda")
    R = tle.LogitRules(n, V, tokens=ids.flatten(), token_start=torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                       repetition=rep)
    out = torch.empty_like(x)
    tle.logits_adjust(out, x, R)
    seen = torch.zeros(n, V, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), True)
    want = torch.where(seen, torch.where(x > 0, x.double() / rep.double()[:, None], x.double() * rep.double()[:, None]), x.double())
    assert bool(((out.double() - want).abs() <= 2.0 ** -23 * want.abs()).all())
    with pytest.raises(tle.TleError):
        tle.logits_adjust(torch.empty(n + 1, 1, device="cuda"), torch.empty(n + 1, 1, device="cuda"), tle.LogitRules(n + 1, 1))


def test_one_mask_for_all_rows(cuda):
    import torch
    import tle
    c = make(5, 700, 60, seed=11, biases=8, mask=True)
    shared = dev(c["allowed"][:1])
    R = tle.LogitRules(5, 700, **{k: dev(c[k]) for k in KEYS if k in c and k != "allowed"}, allowed=shared.expand(5, -1))
    out = torch.empty(5, 700, device="cuda")
    tle.logits_adjust(out, dev(c["x"]), R)
    c["allowed"] = np.repeat(c["allowed"][:1], 5, 0)
    check(c, out)


def test_rules_and_tensors_are_checked(cuda):
    import torch
    import tle
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *x: torch.tensor(x, dtype=torch.float32, device="cuda")  # noqa: E731
    ok = dict(tokens=i32(1, 2, 3), token_start=i32(0, 1, 3), repetition=f32(1, 2))
    tle.LogitRules(2, 50, **ok)
    for bad in (dict(tokens=ok["tokens"].long()), dict(tokens=ok["tokens"].cpu()), dict(token_start=i32(0, 3)),
                dict(token_start=None), dict(tokens=None), dict(repetition=f32(1)), dict(repetition=f32(1, 2).double()),
                dict(tokens=i32(1, 2, 3, 4)[::2]), dict(n_prompt=i32(1, 2, 3)), dict(bias_tokens=i32(1)),
                dict(bias_tokens=i32(1), bias_values=f32(1, 2), bias_start=i32(0, 1, 1)),
                dict(allowed=i32(1, 2)), dict(allowed=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
                dict(allowed=torch.zeros(2, 4, dtype=torch.int32, device="cuda")[:, ::2])):
        with pytest.raises(ValueError):
            tle.LogitRules(2, 50, **{**ok, **bad})
    R = tle.LogitRules(2, 50, **ok)
    x = torch.zeros(2, 50, device="cuda")
    for a, b in ((x[:1], x), (x, x[:, :49]), (x.double(), x), (x, x.cpu()), (torch.zeros(50, 2, device="cuda").T, x),
                 (torch.zeros(1, 50, device="cuda").expand(2, 50), x)):
        with pytest.raises((ValueError, tle.TleError)):
            tle.logits_adjust(a, b, R)


def test_bad_ids_are_skipped_and_reported(cuda):
    import torch
    import tle
    for key in ("tokens", "bias_tokens"):
        for bad in (-1, 700, 1 << 30, -(1 << 31)):
            c = make(3, 700, 90, seed=7, biases=50)
            c[key][[0, 5, -1]] = bad
            out = torch.empty(3, 700, device="cuda")
            tle.logits_adjust(out, dev(c["x"]), rules(c))
            check(c, out)
            assert tle.device_error() == 0x106


def test_starts_outside_the_list_are_cut(cuda):
    """Starts and ends beyond the lists read nothing outside them; a start
    behind its end is an empty list."""
    import torch
    import tle
    c = make(2, 300, 40, seed=8, biases=10)
    nt, nb = c["tokens"].size, c["bias_tokens"].size
    R = rules({**c, "token_start": np.array([-5, nt + 1000, 3], np.int32), "bias_start": np.array([-9, nb + 7, 0], np.int32)})
    out = torch.empty(2, 300, device="cuda")
    tle.logits_adjust(out, dev(c["x"]), R)
    c["token_start"], c["bias_start"] = np.array([0, nt, nt], np.int32), np.array([0, nb, nb], np.int32)
    check(c, out)                  # n_prompt counts from the cut start


def test_strides_stream_and_replay(cuda):
    import torch
    import tle
    c = make(6, 1003, 200, seed=9, biases=20, mask=True)
    wide = torch.full((6, 1200), 7.0, device="cuda")
    wide[:, 100:1103] = dev(c["x"])
    dst = torch.full((6, 1301), 5.0, device="cuda")
    words = torch.full((6, 50), -1, dtype=torch.int32, device="cuda")
    words[:, 3:35] = dev(c["allowed"])
    R = tle.LogitRules(6, 1003, **{k: dev(c[k]) for k in KEYS if k in c and k != "allowed"}, allowed=words[:, 3:35])
    tle.logits_adjust(dst[:, 7:1010], wide[:, 100:1103], R)
    check(c, dst[:, 7:1010])
    assert bool((dst[:, :7] == 5).all()) and bool((dst[:, 1010:] == 5).all())
    first = dst.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    dst.fill_(5)
    side.wait_stream(torch.cuda.current_stream())
    tle.logits_adjust(dst[:, 7:1010], wide[:, 100:1103], R, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tle.logits_adjust(dst[:, 7:1010], wide[:, 100:1103], R)
    wide.mul_(-0.5)
    c["x"] = c["x"] * np.float32(-0.5)
    graph.replay()
    check(c, dst[:, 7:1010])


@pytest.mark.parametrize("far", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 3, 2 ** 31 - 200, 2 ** 30 + 1, -2 ** 31])
def test_starts_far_outside_the_list(cuda, far):
    """Starts and ends next to the largest and smallest 32-bit numbers: both
    ends are cut to the list, whatever its alignment."""
    import torch
    import tle
    c = make(4, 300, 40, seed=13, biases=10)
    nt, nb = c["tokens"].size, c["bias_tokens"].size
    starts, ends = ("token_start", "bias_start"), (nt, nb)
    for at in range(5):                                  # which start is the far one
        given = {k: np.linspace(0, n, 5).astype(np.int32) for k, n in zip(starts, ends)}
        cut = {}
        for k, n in zip(starts, ends):
            given[k][at] = far
            cut[k] = np.clip(given[k], 0, n)
        for shift in range(4):
            room = dev(np.concatenate([np.full(shift, 7, np.int32), c["tokens"]]))
            R = tle.LogitRules(4, 300, **{k: dev(c[k]) for k in KEYS if k in c and k not in starts + ("tokens",)},
                               tokens=room[shift:], **{k: dev(given[k]) for k in starts})
            out = torch.empty(4, 300, device="cuda")
            tle.logits_adjust(out, dev(c["x"]), R)
            # the rows' own lists, one behind the other (a start behind its end: none)
            rows = {}
            for k, lst in zip(starts, (("tokens",), ("bias_tokens", "bias_values"))):
                parts = [slice(cut[k][r], max(cut[k][r], cut[k][r + 1])) for r in range(4)]
                for name in lst:
                    rows[name] = np.concatenate([c[name][p] for p in parts])
                rows[k] = np.concatenate([[0], np.cumsum([p.stop - p.start for p in parts])]).astype(np.int32)
            check({**c, **rows}, out)
    assert tle.device_error() == 0
