"""Attention over 8-bit pages where one team of warps has segments longer than
the ring of tiles: the formula in 64 bits (tolerances as in test_cache8_gpu.py),
and the same bits in many calls, alone and one behind another, also where
sequences share pages, so that some of a CTA's copies come from the cache and others from memory.
"""
import pytest

from test_cache8_gpu import Case, attention64

pytestmark = pytest.mark.gpu

# positions, new tokens, heads, page, CTAs, whether all sequences have the first one's pages
CASES = [
    ([5000], [1], (32, 4), 64, 1, False),                     # four segments of 40 tiles in one CTA
    ([1535], [1], (32, 4), 256, 2, False),                    # 12 tiles, two segments a CTA
    ([2000, 1990], [2, 2], (32, 4), 128, 4, False),           # 16 rows
    ([4000], [4], (32, 4), 64, 2, False),                     # 32 rows
    ([4900, 2100], [1, 3], (32, 4), 64, 2, False),            # 8 and 24 rows in one CTA
    ([2600] * 6, [1] * 6, (32, 4), 64, 6, True),              # shared pages
    ([3000] * 4, [2] * 4, (32, 8), 1024, 8, True),
    ([20000] * 3, [1] * 3, (32, 4), 128, 0, True),            # as the plan has it
]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_segments_longer_than_the_ring(cuda, i, act):
    import torch
    import tle
    pos, new, heads, page, ctas, shared = CASES[i]
    c = Case(pos, new, heads=heads, page=page, act=act, seed=300 + i, max_ctas=ctas)
    if shared:
        c.tables = [c.tables[0]] * len(pos)
        c.batch = tle.PagedChunkBatch(c.cache, c.tables, pos, new, max_ctas=ctas)
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    assert tle.device_error() == 0
    want, tol = attention64(c, c.q)
    assert bool(((c.out[:c.T].double() - want).abs() <= tol).all())
    outs = [torch.empty_like(c.out) for _ in range(25)]
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for j, out in enumerate(outs):
        if j % 5 == 0:
            flush.zero_()                                     # the pools leave the cache
        c.batch.attend(c.q, out, c.layer)
    torch.cuda.synchronize()
    assert all(torch.equal(out[:c.T], c.out[:c.T]) for out in outs)
    assert tle.device_error() == 0
