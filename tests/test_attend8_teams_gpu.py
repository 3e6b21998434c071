"""Attention over 8-bit pages where one CTA has many segments, by max_ctas: its
warps then work in teams, on several segments at once.  Against the formula in
64 bits (tolerances as in test_cache8_gpu.py), and the same bits every time.
"""
import pytest

from test_cache8_gpu import Case, attention64

pytestmark = pytest.mark.gpu

# positions, new tokens, heads, page, CTAs
CASES = [
    ([60] * 9, [1] * 9, (32, 4), 64, 1),                              # 36 segments of a tile
    ([5, 200, 0, 130, 400, 64, 127, 128], [1] * 8, (8, 8), 64, 2),    # one to four tiles
    ([300, 2, 200], [1, 3, 2], (12, 4), 128, 1),
    ([100] * 11 + [5000] + [90] * 3, [1] * 15, (8, 2), 64, 1),        # one longer than the ring among short ones
    ([5000] + [30] * 30, [1] * 31, (4, 1), 256, 1),                   # at the start
    ([30] * 20 + [4000, 20], [1] * 22, (4, 1), 64, 1),                # at the end
    ([1000, 1200, 900, 1100], [1] * 4, (32, 4), 64, 2),               # two teams
    ([700, 1500, 650, 2047, 900], [2] * 5, (32, 4), 128, 2),          # with 16 rows
    ([1000, 1200, 900, 1100], [4] * 4, (32, 4), 64, 2),               # 32 rows
    ([200, 100, 300, 50, 400], [4] * 5, (32, 4), 64, 1),              # 32 rows, three teams
    ([200, 100, 300, 50, 400, 260], [1, 4, 2, 3, 1, 4], (32, 4), 64, 1),
    ([0] * 40, [1] * 40, (32, 4), 64, 3),                             # nothing but the new row
    ([64, 0, 500, 0], [1, 0, 1, 0], (32, 8), 64, 1),                  # sequences without new tokens
    ([600] * 30, [1] * 30, (32, 4), 64, 4),                           # 30 segments a CTA, more than are held at once
]


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_teams(cuda, i, act):
    import torch
    import tle
    pos, new, heads, page, ctas = CASES[i]
    c = Case(pos, new, heads=heads, page=page, act=act, seed=200 + i, max_ctas=ctas)
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    assert tle.device_error() == 0
    want, tol = attention64(c, c.q)
    assert bool(((c.out[:c.T].double() - want).abs() <= tol).all())
    again = torch.empty_like(c.out)
    for _ in range(5):
        c.batch.attend(c.q, again, c.layer)
        assert torch.equal(again[:c.T], c.out[:c.T])
    assert tle.device_error() == 0


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_teams_bad_pages_and_replays(cuda, act):
    """Pages outside the pool count as zeros with several teams too; a graph gives the call's bits."""
    import torch
    import tle
    pos = [100, 300, 64, 500, 10, 250, 90]
    c = Case(pos, [1] * 7, heads=(32, 4), act=act, seed=230, max_ctas=1)
    good = torch.empty_like(c.out)
    c.batch.attend(c.q, good, c.layer)
    keep = c.tables[3].clone()
    c.tables[3][2] = c.cache.n_pages + 5
    c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    assert tle.device_error(clear=True) == 0x105
    same = [0, 1, 2, 4, 5, 6]
    assert torch.equal(c.out[same], good[same]) and not torch.equal(c.out[3], good[3]) and bool(torch.isfinite(c.out[:7]).all())
    c.tables[3].copy_(keep)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.batch.attend(c.q, c.out, c.layer)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.batch.attend(c.q, c.out, c.layer)
    for _ in range(3):
        c.out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out[:7], good[:7])
    assert tle.device_error() == 0
