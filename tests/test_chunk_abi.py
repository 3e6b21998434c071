"""CPU tests of the chunk calls and the logit rules: the work plan of
tle_chunk_desc_paged covers every K/V tile of every row block once, and bad
arguments are refused before any device work (fake, never dereferenced
pointers)."""
import ctypes

import numpy as np
import pytest

import tle

TILE, ITEM, FEW = 128, 256, 32
P = 0x400000


def describe(pos, new, heads=(32, 4), page=64, max_ctas=0, n_pages=None, table=lambda i: 0x4000 * (i + 1)):
    n = len(pos)
    shape = tle.Shape(2, heads[0], heads[1], 64, 10000.0)
    c = (tle.PagedChunk * max(n, 1))()
    for i in range(n):
        c[i] = tle.PagedChunk(table(i), -(-(pos[i] + new[i]) // page) if n_pages is None else n_pages[i], pos[i], new[i], 0)
    plan = tle.ChunkPlan()
    nbytes = tle.lib().tle_chunk_desc_bytes(ctypes.byref(shape), c, n, max_ctas)
    if nbytes == 0:
        return tle.TLE_ERR_INVALID, None, plan
    buf = np.zeros((nbytes + 7) // 8, np.int64)
    rc = tle.lib().tle_chunk_desc_paged(ctypes.byref(shape), page, c, n, max_ctas, buf.ctypes.data, nbytes,
                                        ctypes.byref(plan))
    assert rc != 0 or plan.desc_bytes <= nbytes
    return rc, buf.view(np.uint8)[:plan.desc_bytes], plan


def parse(buf, plan):
    b, at = buf.tobytes(), 32

    def take(count, width, dtype=np.int32):
        nonlocal at
        a = np.frombuffer(b[at:at + count * width], dtype).reshape(count, width // 4)
        at += count * width
        return a
    cta = take(plan.n_ctas + plan.n_few_ctas, 64)
    segs = take(plan.n_segs, 64)
    seqs = take(plan.n_seqs, 24)
    merges = take(plan.n_merge, 24)
    toks = take(plan.n_tokens, 8)
    assert at == len(b)
    return seqs, segs, merges, toks, cta


PAGES, POS, FIRST, KVH, ROW0, ROWS, T0, T1, PART, POS_MIN, KV_LEN, SEG0, SEG1, SEQ = 0, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14


@pytest.mark.parametrize("seed", range(12))
def test_plan_covers_every_tile_once(seed):
    r = np.random.default_rng(seed)
    n = int(r.integers(1, 60 if seed % 2 else 4))
    pos = [int(x) for x in r.integers(0, 5000, n)]
    new = [int(x) for x in r.integers(0, [2, 40, 700][seed % 3], n)]
    heads = [(32, 4), (8, 8), (20, 4), (7, 1)][seed % 4]
    check_plan(pos, new, heads, [0, 1, 3, 148][int(r.integers(0, 4))])


@pytest.mark.parametrize("pos,new,heads", [
    ([0, 9], [40000, 5], (32, 4)),                       # more items than are sorted
    ([500] * 300, [1] * 300, (32, 32)),                  # the same of few rows
    ([1 << 20, 5], [1, 300], (32, 4)),                   # one item far longer than the others
])
def test_plan_of_many_or_uneven_items(pos, new, heads):
    check_plan(pos, new, heads, 0)


def check_plan(pos, new, heads, max_ctas):
    n = len(pos)
    rc, buf, plan = describe(pos, new, heads, max_ctas=max_ctas)
    assert rc == 0, tle.lib().tle_last_error()
    g = heads[0] // heads[1]
    seqs, segs, merges, toks, cta = parse(buf, plan)
    assert plan.n_tokens == sum(new) and plan.n_seqs == n
    assert [tuple(x) for x in toks] == [(s, pos[s] + t) for s in range(n) for t in range(new[s])]
    first = np.cumsum([0] + new)[:-1]
    assert np.array_equal(seqs[:, 3], pos) and np.array_equal(seqs[:, 4], new) and np.array_equal(seqs[:, 5], first)
    assert max(plan.n_ctas, plan.n_few_ctas) <= (max_ctas or 148)
    assert cta.shape[0] == 0 or (cta[0, SEG0] == 0 and cta[-1, SEG1] == plan.n_segs)
    assert np.array_equal(cta[1:, SEG0], cta[:-1, SEG1]) and np.all(cta[:, SEG0] <= cta[:, SEG1])
    for x in cta[cta[:, SEG0] < cta[:, SEG1]]:                         # a copy of the CTA's first piece
        assert np.array_equal(np.delete(x, [SEG0, SEG1]), np.delete(segs[x[SEG0]], [SEG0, SEG1]))
    few0 = cta[plan.n_ctas, SEG0] if plan.n_few_ctas else plan.n_segs
    chunk_rows = np.array(new)[segs[:, SEQ]] * g                       # chunks of many rows, then of few
    assert np.all(chunk_rows[:few0] > FEW) and np.all(chunk_rows[few0:] <= FEW)
    assert np.array_equal(segs[:, POS], np.array(pos)[segs[:, SEQ]]) and np.array_equal(segs[:, FIRST], first[segs[:, SEQ]])
    assert np.array_equal(segs[:, PAGES], 0x4000 * (segs[:, SEQ] + 1))
    assert np.array_equal(segs[:, POS_MIN], segs[:, POS] + segs[:, ROW0] // g)
    assert np.array_equal(segs[:, KV_LEN], segs[:, POS] + (segs[:, ROW0] + segs[:, ROWS] - 1) // g + 1)
    items = {(s, h, r0): rows for s, h, r0, rows in segs[:, [SEQ, KVH, ROW0, ROWS]]}
    starts = {}                                                        # blocks of rows, each row in one
    for s, h, r0 in sorted(items):
        at = starts.get((s, h), 0)
        assert r0 == at and r0 % (ITEM // 2) == 0 and 0 < items[(s, h, r0)] <= ITEM
        starts[(s, h)] = at + items[(s, h, r0)]
    assert starts == {(s, h): new[s] * g for s in range(n) for h in range(heads[1]) if new[s]}
    seen, parts = {k: [] for k in items}, {}
    used = np.zeros(plan.part_rows, int)
    for s, h, r0, rows, t0, t1, part in segs[:, [SEQ, KVH, ROW0, ROWS, T0, T1, PART]]:
        assert items[(s, h, r0)] == rows and t0 < t1
        seen[(s, h, r0)].append((t0, t1))
        if part >= 0:
            used[part:part + rows] += 1
            parts.setdefault((s, h, r0), []).append(part)
    for (s, h, r0), rows in items.items():
        tiles = (pos[s] + (r0 + rows - 1) // g) // TILE + 1
        cuts = seen[(s, h, r0)]
        cuts.sort()
        assert cuts[0][0] == 0 and cuts[-1][1] == tiles                # without gaps
        assert all(a[1] == b[0] for a, b in zip(cuts, cuts[1:]))
        assert len(cuts) == 1 or (s, h, r0) in parts                   # alone: it writes the result itself
    assert np.all(used == 1)
    merged = {}
    for s, h, r0, rows, part, k in merges:
        assert items[(s, h, r0)] == rows and rows <= plan.merge_rows and k > 1
        merged[(s, h, r0)] = (part, k)
    assert set(merged) == set(parts)
    for key, lst in parts.items():                                     # a block of partial rows per part, in order
        part, k = merged[key]
        assert lst == [part + j * items[key] for j in range(k)] and k == len(seen[key])


def test_plan_balances_long_work():
    """A prompt piece late in a long context: no CTA has more than a few
    tiles above the even share."""
    rc, buf, plan = describe([30000], [2048])
    assert rc == 0
    _, segs, _, _, cta = parse(buf, plan)
    cost = [sum(2 * (x[T1] - x[T0]) for x in segs[a:b]) for a, b in cta[:, [SEG0, SEG1]]]
    assert plan.n_ctas == 148 and max(cost) <= sum(cost) / 148 + 16


def test_desc_buffer_size_and_plan_number():
    """A buffer of the stated size does at any positions, a smaller one than
    needed is refused; the number that the calls check differs between plans."""
    shape = tle.Shape(2, 32, 4, 64, 10000.0)
    c, plan, numbers = (tle.PagedChunk * 3)(), tle.ChunkPlan(), set()
    for pos in ([0, 0, 0], [5000, 1, 300], [5001, 1, 300], [9000, 9000, 9000]):
        for i, new in enumerate((300, 1, 20)):
            c[i] = tle.PagedChunk(0x4000, 500, pos[i], new, 0)
        nbytes = tle.lib().tle_chunk_desc_bytes(ctypes.byref(shape), c, 3, 0)
        buf = np.zeros(nbytes // 8 + 1, np.int64)
        go = lambda size, at=0: tle.lib().tle_chunk_desc_paged(  # noqa: E731
            ctypes.byref(shape), 64, c, 3, 0, buf.ctypes.data + at, size, ctypes.byref(plan))
        assert go(nbytes) == tle.TLE_OK and go(plan.desc_bytes) == tle.TLE_OK
        numbers.add((int(buf[0]), plan.n_segs, plan.n_merge, plan.part_rows, plan.n_ctas, plan.n_few_ctas))
        assert go(plan.desc_bytes - 1) == tle.TLE_ERR_INVALID and go(plan.desc_bytes, 4) == tle.TLE_ERR_INVALID
    assert len({x[0] for x in numbers}) == len({x[1:] for x in numbers}) > 1


def test_empty_batches():
    rc, buf, plan = describe([5, 0], [0, 0], table=lambda i: 0)
    assert rc == 0 and plan.n_tokens == 0 and plan.n_segs == 0 and plan.part_rows == 0
    assert tle.lib().tle_prefill_bf16_paged_workspace_bytes(ctypes.byref(plan)) == 0


@pytest.mark.parametrize("kw,what", [
    (dict(pos=[-1], new=[3]), "pos"), (dict(pos=[0], new=[-1]), "n_tokens"),
    (dict(pos=[60], new=[5], n_pages=[1]), "n_pages * page_rows"),
    (dict(pos=[0], new=[5], table=lambda i: 0), "page table"),
    (dict(pos=[0], new=[5], table=lambda i: 0x4002), "aligned"),
    (dict(pos=[0], new=[5], page=48), "power of two"), (dict(pos=[0], new=[5], page=8), "power of two"),
    (dict(pos=[], new=[]), "n_seqs"), (dict(pos=[2147483000], new=[600], n_pages=[1 << 30]), "too long"),
    (dict(pos=[0], new=[5], heads=(9, 2)), "multiple"), (dict(pos=[0], new=[5], heads=(129, 1)), "multiple"),
    (dict(pos=[0], new=[5], heads=(0, 1)), "shape"),
])
def test_desc_refuses(kw, what):
    rc, _, _ = describe(**kw)
    assert rc != tle.TLE_OK
    assert what in tle.lib().tle_last_error().decode()


def call(name, plan, shape=None, pool=None, q=P, qs=2048, k=P, ks=256, v=P, vs=256, qo=P, act=0, layer=0, flags=1,
         desc=P, ws=P, wsb=1 << 30, out=P, os=2048):
    L = tle.lib()
    shape = shape or tle.Shape(2, 32, 4, 64, 10000.0)
    if pool is None:
        pool = tle.PagePool(P, P, 100, 64) if name == "tle_append_paged" else tle.PagePoolBf16(P, P, 100, 64)
    pp = ctypes.addressof(pool) if pool else None
    if name.startswith("tle_append"):
        return getattr(L, name)(ctypes.byref(shape), pp, ctypes.byref(plan), desc, q, qs, k, ks, v, vs, qo, act, layer,
                                flags, None)
    return L.tle_prefill_bf16_paged(ctypes.byref(shape), pp, ctypes.byref(plan), desc, q, qs, out, os, act, layer, ws,
                                    wsb, None)


@pytest.mark.parametrize("name", ["tle_append_paged", "tle_append_bf16_paged", "tle_prefill_bf16_paged"])
def test_calls_refuse_bad_arguments(name):
    _, _, plan = describe([3000], [40])
    assert plan.part_rows > 0
    bad = tle.TLE_ERR_INVALID
    pools = tle.PagePool if name == "tle_append_paged" else tle.PagePoolBf16
    assert call(name, plan, pool=False) == bad
    assert call(name, plan, pool=pools(P, None, 100, 64)) == bad
    assert call(name, plan, pool=pools(P, P + 8, 100, 64)) == bad
    assert call(name, plan, pool=pools(P, P, 0, 64)) == bad
    assert call(name, plan, pool=pools(P, P, 100, 128)) == bad          # the plan is for pages of 64
    assert call(name, plan, pool=pools(P, P, 1 << 30, 64)) == bad
    assert call(name, plan, shape=tle.Shape(2, 16, 4, 64, 10000.0)) == bad
    assert call(name, plan, shape=tle.Shape(2, 32, 4, 128, 10000.0)) == tle.TLE_ERR_UNSUPPORTED
    assert call(name, plan, shape=tle.Shape(0, 32, 4, 64, 10000.0)) == bad
    assert call(name, plan, layer=2) == bad and call(name, plan, layer=-1) == bad
    assert call(name, plan, act=2) == tle.TLE_ERR_UNSUPPORTED
    assert call(name, plan, desc=None) == bad and call(name, plan, desc=P + 8) == bad
    assert call(name, plan, q=P + 4) == bad
    assert call(name, plan, qs=2047) == bad and call(name, plan, qs=2052) == bad
    if name == "tle_prefill_bf16_paged":
        assert call(name, plan, q=None) == bad and call(name, plan, out=None) == bad
        assert call(name, plan, os=2040) == bad
        assert call(name, plan, ws=None) == tle.TLE_ERR_WORKSPACE
        assert call(name, plan, wsb=1024) == tle.TLE_ERR_WORKSPACE
        assert call(name, plan, ws=P + 4) == bad
    else:
        assert call(name, plan, q=None) == bad and call(name, plan, qo=None) == bad
        assert call(name, plan, qs=2056) == bad                         # q in place, with another stride
        assert call(name, plan, k=None) == bad and call(name, plan, v=P + 2) == bad
        assert call(name, plan, ks=248) == bad and call(name, plan, vs=260) == bad
        assert call(name, plan, flags=2) == bad
    _, _, small = describe([3000], [40], page=16)
    if name != "tle_append_paged":                                      # bf16 pools: pages of 64 rows at least
        assert call(name, small, pool=pools(P, P, 1000, 16)) == bad


def test_calls_without_tokens_do_nothing():
    _, _, plan = describe([5], [0])
    for name in ("tle_append_paged", "tle_append_bf16_paged", "tle_prefill_bf16_paged"):
        assert call(name, plan, q=None, k=None, v=None, qo=None, out=None, ws=None, wsb=0) == tle.TLE_OK


def test_logit_rules_refuse_bad_arguments():
    L = tle.lib()

    def go(out=P, os=100, x=P, xs=100, n=2, V=100, **kw):
        r = tle.LogitRulesDesc(**kw)
        return L.tle_logits_adjust(out, os, x, xs, n, V, ctypes.byref(r), None)
    bad = tle.TLE_ERR_INVALID
    assert go(out=None) == bad and go(x=None) == bad and go(n=0) == bad and go(V=0) == bad and go(n=65536) == bad
    assert go(os=99) == bad and go(xs=99) == bad and go(os=104) == bad
    assert go(tokens=P) == bad and go(repetition=P) == bad and go(presence=P, token_start=P) == bad
    assert go(bias_tokens=P) == bad and go(bias_tokens=P, bias_values=P) == bad
    assert go(allowed=P, allowed_stride=3) == bad and go(allowed=P, allowed_stride=-4) == bad
    assert go(out=P + 2) == bad and go(x=P + 1) == bad and go(tokens=P + 2, token_start=P, frequency=P) == bad
    assert go(tokens=P, token_start=P, frequency=P + 2) == bad and go(allowed=P + 2, allowed_stride=4) == bad
    assert go(tokens=P, token_start=P, n_tokens=(1 << 30) + 1) == bad
    assert go(tokens=P, token_start=P, n_tokens=-1) == bad
    assert L.tle_logits_adjust(P, 100, P, 100, 2, 100, None, None) == bad


def test_attention_in_place_wants_one_stride():
    """out = q with another stride would overwrite rows of q that other CTAs
    still read: refused before any launch."""
    _, _, plan = describe([3000], [40])
    assert call("tle_prefill_bf16_paged", plan, os=2056) == tle.TLE_ERR_INVALID
    assert "stride" in tle.lib().tle_last_error().decode()
    assert call("tle_prefill_bf16_paged", plan, qs=4096) == tle.TLE_ERR_INVALID


@pytest.mark.parametrize("pos,new", [([3000, 10, 5], [40, 1, 300]), ([0], [1]), ([20], [0])])
def test_descriptor_at_any_8_byte_boundary(pos, new):
    """The records are stored without alignment beyond the buffer's 8 bytes:
    the same bytes at 0 and at 8 modulo 16."""
    shape, n = tle.Shape(2, 32, 4, 64, 10000.0), len(pos)
    c = (tle.PagedChunk * n)(*[tle.PagedChunk(0x4000, 500, p, m, 0) for p, m in zip(pos, new)])
    nbytes = tle.lib().tle_chunk_desc_bytes(ctypes.byref(shape), c, n, 0)
    got = []
    for off in (0, 8):
        raw = np.full(nbytes + 64, 0xAB, np.uint8)
        at = (-raw.ctypes.data) % 16 + off
        plan = tle.ChunkPlan()
        assert tle.lib().tle_chunk_desc_paged(ctypes.byref(shape), 64, c, n, 0, raw.ctypes.data + at, nbytes, ctypes.byref(plan)) == 0
        assert np.all(raw[:at] == 0xAB) and np.all(raw[at + plan.desc_bytes:] == 0xAB)
        got.append(raw[at:at + plan.desc_bytes].copy())
    assert np.array_equal(got[0], got[1])
