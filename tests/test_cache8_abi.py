"""CPU tests of the appends by rules and the 8-bit page calls: refusals before
any device work (fake, never dereferenced pointers), workspace sizes, and the
frequencies for long contexts."""
import ctypes

import numpy as np
import pytest

import tle

P = 0x400000


def describe(pos, new, heads=(32, 4), page=64):
    shape, n = tle.Shape(2, heads[0], heads[1], 64, 10000.0), len(pos)
    c = (tle.PagedChunk * n)(*[tle.PagedChunk(0x4000, 1 << 20, p, m, 0) for p, m in zip(pos, new)])
    plan, nbytes = tle.ChunkPlan(), tle.lib().tle_chunk_desc_bytes(ctypes.byref(shape), c, n, 0)
    buf = np.zeros(nbytes // 8 + 1, np.int64)
    assert tle.lib().tle_chunk_desc_paged(ctypes.byref(shape), page, c, n, 0, buf.ctypes.data, nbytes, ctypes.byref(plan)) == 0
    return shape, c, plan


def workspace(shape, c, plan, n=None):
    return tle.lib().tle_prefill_q8_paged_workspace_bytes(ctypes.byref(shape), c, len(c) if n is None else n, ctypes.byref(plan))


def test_workspace_sizes():
    shape, c, plan = describe([100, 40], [1, 4])            # few rows only: the partial results
    assert workspace(shape, c, plan) == (tle.lib().tle_prefill_bf16_paged_workspace_bytes(ctypes.byref(plan)) + 15) // 16 * 16
    shape, c, plan = describe([100, 40, 300], [28, 4, 5])   # 128 and 305 rows: 1 + 3 pages of 128
    size = workspace(shape, c, plan)
    assert size >= 4 * (2 * 128 * 256 * 2 + 4) + 32 + 64 * plan.n_segs
    assert size <= 4 * (2 * 128 * 256 * 2 + 4) + 128 + 64 * (plan.n_segs + plan.n_ctas + plan.n_few_ctas) + 260 * plan.part_rows
    assert workspace(shape, c, plan, 2) == 0 and "plan" in tle.lib().tle_last_error().decode()


def pool(**kw):
    d = dict(key_codes=P, value_codes=P, key_scale=P, value_scale=P, n_pages=100, page_rows=64)
    d.update(kw)
    return tle.PagePoolQ8(*d.values())


def rules(**kw):
    d = dict(layout=0, rotary_dim=64, inv_freq=None, rope_factor=1.0, norm_eps=0.0, q_norm=None, k_norm=None)
    d.update(kw)
    return tle.AppendRulesDesc(*d.values())


BAD = tle.TLE_ERR_INVALID


@pytest.mark.parametrize("name", ["tle_append_q8_paged", "tle_append_rules_paged", "tle_append_rules_bf16_paged"])
def test_appends_refuse_bad_arguments(name):
    shape, _, plan = describe([3000], [40])
    pools = {"tle_append_q8_paged": pool(), "tle_append_rules_paged": tle.PagePool(P, P, 100, 64),
             "tle_append_rules_bf16_paged": tle.PagePoolBf16(P, P, 100, 64)}

    def go(pl=pools[name], r=None, q=P, qs=2048, k=P, ks=256, v=P, vs=256, qo=P, act=0, layer=0, flags=1, desc=P, shape=shape):
        return getattr(tle.lib(), name)(ctypes.byref(shape), ctypes.addressof(pl) if pl else None, ctypes.byref(plan), desc, q, qs, k, ks,
                                        v, vs, qo, act, layer, flags, ctypes.addressof(r) if r else None, None)
    assert go(pl=None) == BAD and go(desc=None) == BAD and go(layer=2) == BAD and go(flags=2) == BAD
    assert go(q=None) == BAD and go(qo=None) == BAD and go(qs=2052) == BAD and go(k=P + 4) == BAD and go(vs=248) == BAD
    assert go(act=2) == tle.TLE_ERR_UNSUPPORTED
    assert go(r=rules(layout=2)) == BAD and go(r=rules(norm_eps=-1.0)) == BAD and go(r=rules(norm_eps=float("nan"))) == BAD
    assert go(r=rules(rotary_dim=24)) == tle.TLE_ERR_UNSUPPORTED and go(r=rules(rotary_dim=80)) == tle.TLE_ERR_UNSUPPORTED
    assert go(r=rules(rotary_dim=0)) == tle.TLE_ERR_UNSUPPORTED
    assert go(r=rules(q_norm=P + 2)) == BAD and go(r=rules(k_norm=P + 1)) == BAD and go(r=rules(inv_freq=P + 2)) == BAD
    if name == "tle_append_q8_paged":
        for kw in (dict(key_codes=None), dict(value_codes=P + 8), dict(key_scale=None), dict(value_scale=None), dict(key_scale=P + 8),
                   dict(n_pages=0), dict(page_rows=128), dict(page_rows=32), dict(n_pages=1 << 30)):
            assert go(pl=pool(**kw)) == BAD


def test_read_refuses_bad_arguments():
    shape, _, plan = describe([3000], [40])

    def go(pl=pool(), k=P, ks=256, v=P, vs=256, n=3040, t=0, layer=0, flags=0, desc=P):
        return tle.lib().tle_read_q8_paged(ctypes.byref(shape), ctypes.addressof(pl) if pl else None, ctypes.byref(plan), desc, k, ks, v, vs,
                                           n, t, layer, flags, None)
    assert go(pl=None) == BAD and go(pl=pool(key_scale=None)) == BAD and go(pl=pool(page_rows=128)) == BAD
    assert go(desc=None) == BAD and go(desc=P + 8) == BAD and go(layer=-1) == BAD and go(t=2) == tle.TLE_ERR_UNSUPPORTED
    assert go(k=P + 8) == BAD and go(ks=250) == BAD and go(vs=252) == BAD and go(n=-1) == BAD and go(flags=2) == BAD
    assert go(flags=1) == BAD                              # 40 new tokens, not 3040
    assert go(n=0) == 0 and go(k=None, v=None) == 0


def test_attention_refuses_bad_arguments():
    shape, c, plan = describe([3000], [40])
    size = workspace(shape, c, plan)

    def go(pl=pool(), q=P, qs=2048, out=P, os=2048, act=0, layer=0, ws=P, wsb=size, desc=P, plan=plan):
        return tle.lib().tle_prefill_q8_paged(ctypes.byref(shape), ctypes.addressof(pl) if pl else None, ctypes.byref(plan), desc, q, qs, out,
                                              os, act, layer, ws, wsb, None)
    assert go(pl=None) == BAD and go(pl=pool(value_scale=None)) == BAD and go(pl=pool(key_codes=P + 4)) == BAD
    assert go(q=None) == BAD and go(out=P + 8) == BAD and go(os=2056) == BAD and go(qs=2040) == BAD and go(desc=P + 4) == BAD
    assert go(act=3) == tle.TLE_ERR_UNSUPPORTED and go(layer=2) == BAD
    assert go(ws=None) == tle.TLE_ERR_WORKSPACE and go(wsb=100000) == tle.TLE_ERR_WORKSPACE and go(ws=P + 8) == BAD
    _, _, none = describe([5], [0])
    assert go(plan=none, q=None, out=None, ws=None, wsb=0) == 0


def test_rope_frequencies():
    base = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    f, m = tle.rope_frequencies()
    assert m == 1.0 and np.allclose(f, base, rtol=2.0 ** -23)
    f, m = tle.rope_frequencies(32, 500000.0, "linear", 4.0)
    assert m == 1.0 and np.allclose(f, 500000.0 ** (-np.arange(0, 32, 2) / 32) / 4, rtol=2.0 ** -23)
    f, m = tle.rope_frequencies(64, 10000.0, "ntk", 8.0)
    assert m == 1.0 and f[0] == 1.0 and np.isclose(f[-1], base[-1] / 8, rtol=1e-6)      # the slowest pair: as linear
    f, m = tle.rope_frequencies(64, 10000.0, "yarn", 4.0, 2048)
    turns = base * 2048 / (2 * np.pi)
    assert np.isclose(m, 1 + 0.1 * np.log(4)) and np.allclose(np.array(f)[turns > 40], base[turns > 40], rtol=1e-6)
    assert np.allclose(np.array(f)[turns < 0.7], base[turns < 0.7] / 4, rtol=1e-6)
    assert np.all(np.diff(f) < 0) and np.all(np.array(f) <= base * (1 + 1e-6)) and np.all(np.array(f) >= base / 4 * (1 - 1e-6))
    for kw in (dict(rotary_dim=24), dict(rotary_dim=0), dict(rotary_dim=80), dict(base=1.0), dict(scaling="yarn", factor=0.9),
               dict(scaling="linear", factor=float("nan")), dict(scaling="yarn", factor=2.0, original_ctx=0)):
        with pytest.raises(tle.TleError):
            tle.rope_frequencies(**kw)


def test_sampling_refuses_bad_arguments():
    def go(out=P, x=P, xs=100, n=2, V=100, u=P, rules=True, **kw):
        r = tle.SampleRulesDesc(**kw)
        return tle.lib().tle_sample_rows(out, x, xs, n, V, ctypes.byref(r) if rules else None, u, None)
    assert go(out=None) == BAD and go(x=None) == BAD and go(u=None) == BAD and go(rules=False) == BAD
    assert go(n=0) == BAD and go(n=65536) == BAD and go(V=0) == BAD and go(xs=99) == BAD and go(xs=-100) == BAD
    assert go(out=P + 2) == BAD and go(x=P + 1) == BAD and go(u=P + 2) == BAD
    for name in ("temperature", "top_k", "top_p", "min_p"):
        assert go(**{name: P + 2}) == BAD
    assert go(V=262145, xs=262145) == tle.TLE_ERR_UNSUPPORTED
