"""A serving step out of its parts: appends by rules into 8-bit pages, the
attention over them, the logit rules and a token for each row, the token going
into the next step.

Each part is checked against the formula in 64 bits on what it was given
(tolerances as in test_cache8_gpu.py, borders as in test_sample_gpu.py); the
whole step, captured and replayed, gives what it gave when it was called.
"""
import numpy as np
import pytest

from test_cache8_gpu import HD, Case, attention64
from test_sample_gpu import oracle

pytestmark = pytest.mark.gpu

VOCAB, LAYERS = 5003, 2


class Model:
    """Two layers of attention between an embedding and an output matrix, and a batch of sequences in it."""

    def __init__(self, act, heads, page, prompts):
        import torch
        import tle
        self.c = c = Case([0] * len(prompts), prompts, heads=heads, page=page, act=act, layers=LAYERS, seed=41, spare=40)
        H, KH = heads
        n = len(prompts)
        # every sequence gets a page more than its prompt needs, for its next tokens
        ids = torch.randperm(c.cache.n_pages, generator=c.g, device="cuda").to(torch.int32)
        need = [-(-p // page) + 1 for p in prompts]
        c.tables = list(torch.split(ids[:sum(need)].clone(), need))
        c.batch = tle.PagedChunkBatch(c.cache, c.tables, [0] * n, prompts)
        rnd = lambda *d: torch.randn(d, generator=c.g, device="cuda")  # noqa: E731
        self.embed, self.unembed = rnd(VOCAB, H * HD), rnd(H * HD, VOCAB) * (4.0 / (H * HD) ** 0.5)
        self.w = [[rnd(H * HD, m * HD) * (H * HD) ** -0.5 for m in (H, KH, KH)] for _ in range(LAYERS)]
        freq, factor = tle.rope_frequencies(32, scaling="yarn", factor=2.0)
        self.rules = [tle.AppendRules("half", inv_freq=freq, rope_factor=factor, q_norm=torch.rand(HD, device="cuda") + 0.5,
                                      k_norm=torch.rand(HD, device="cuda") + 0.5) for _ in range(LAYERS)]
        words = torch.full((n, (VOCAB + 31) // 32), -1, dtype=torch.int32, device="cuda")
        words[0] = 0x0F0F0F0F
        bias = [torch.tensor(x, device="cuda") for x in ([5, 9] * n, [1.5, -2.0] * n)]
        start = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
        self.logit_rules = tle.LogitRules(n, VOCAB, bias_tokens=bias[0].int(), bias_values=bias[1], bias_start=start, allowed=words)
        f = lambda *x: torch.tensor((x * n)[:n], device="cuda")  # noqa: E731
        self.T, self.k, self.p = f(0.8, 1.2, 0.0), f(40, 0, 7).int(), f(0.95, 0.9, 1.0)
        self.sample_rules = tle.SampleRules(n, VOCAB, self.T, self.k, self.p)
        self.uniform = torch.rand(n, generator=c.g, device="cuda")
        self.logits, self.adjusted = torch.empty(n, VOCAB, device="cuda"), torch.empty(n, VOCAB, device="cuda")
        self.tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.act = c.q.dtype

    def step(self, tokens, last, check=None):
        """tokens of all chunks -> self.tokens, one for each row `last`."""
        import torch
        import tle
        b = self.c.batch
        x = self.embed[tokens]
        for i in range(LAYERS):
            q, k, v = ((x @ w).to(self.act) for w in self.w[i])
            out = torch.empty_like(q)
            b.run(q, k, v, out, i, rules=self.rules[i])
            if check:
                check(i, q, k, v, out)
            x = x + out.float()
        torch.mm(x[last] / (1 + LAYERS) ** 0.5, self.unembed, out=self.logits)
        tle.logits_adjust(self.adjusted, self.logits, self.logit_rules)
        tle.sample_rows(self.tokens, self.adjusted, self.sample_rules, self.uniform)

    def check_layer(self, i, q, k, v, out):
        import torch
        c = self.c
        c.layer = i
        turned = torch.empty_like(q)
        c.batch.append(q, k, v, i, q_out=turned, rules=self.rules[i])   # the same rows once more
        want, tol = attention64(c, turned)
        assert bool(((out.double() - want).abs() <= tol).all())

    def check_tokens(self):
        x, got = self.adjusted.cpu().numpy(), self.tokens.cpu().numpy()
        for r in range(len(got)):
            want, near = oracle(x[r], float(self.T[r]), int(self.k[r]), float(self.p[r]), 0.0, float(self.uniform[r]))
            assert got[r] == want or near <= 2 * VOCAB * 2.0 ** -41 + 2.0 ** -45
            if r == 0:
                assert (got[r] & 7) < 4   # the mask's words leave the lower half of every byte


@pytest.mark.parametrize("act,heads,page,prompts", [
    ("f32", (32, 4), 64, [150, 1, 33]),
    ("bf16", (32, 4), 128, [3, 300, 70]),
    ("bf16", (8, 8), 64, [40, 64, 65, 1, 17]),
    ("f32", (12, 4), 256, [500]),
])
def test_a_prompt_then_tokens(cuda, act, heads, page, prompts):
    import torch
    import tle
    m = Model(act, heads, page, prompts)
    c, n = m.c, len(prompts)
    tokens = torch.randint(0, VOCAB, (sum(prompts),), generator=c.g, device="cuda")
    last = torch.cumsum(torch.tensor(prompts, device="cuda"), 0) - 1
    m.step(tokens, last, m.check_layer)
    m.check_tokens()
    pos = list(prompts)
    every = torch.arange(n, device="cuda")
    for _ in range(4):
        tokens = m.tokens.long().clone()
        assert bool(((tokens >= 0) & (tokens < VOCAB)).all())
        c.pos, c.new, c.T = list(pos), [1] * n, n
        c.batch.set_positions(pos, [1] * n)
        m.uniform.uniform_(generator=c.g)
        m.step(tokens, every, m.check_layer)
        m.check_tokens()
        pos = [p + 1 for p in pos]
    assert tle.device_error() == 0


def test_a_captured_step(cuda):
    """The step as a graph: the same tokens and pages as the calls, at every replay, and under new tokens and numbers."""
    import torch
    import tle
    m = Model("bf16", (32, 4), 64, [100, 9, 300])
    c = m.c
    tokens = torch.randint(0, VOCAB, (409,), generator=c.g, device="cuda")
    m.step(tokens, torch.tensor([99, 108, 408], device="cuda"))
    pools = (c.cache.key_pool, c.cache.key_scale, c.cache.value_pool, c.cache.value_scale)
    before = [t.clone() for t in pools]
    every = torch.arange(3, device="cuda")
    c.batch.set_positions([100, 9, 300], [1, 1, 1])
    fed = m.tokens.long().clone()
    cases = [(fed.clone(), m.uniform.clone())] + [(torch.randint(0, VOCAB, (3,), generator=c.g, device="cuda"),
                                                   torch.rand(3, generator=c.g, device="cuda")) for _ in range(3)]
    want = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t, u in cases:
            fed.copy_(t), m.uniform.copy_(u)
            m.step(fed, every)
            want.append([m.tokens.clone(), m.adjusted.clone()] + [x.clone() for x in pools])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.step(fed, every)
    for (t, u), w in list(zip(cases, want)) * 2:
        for x, y in zip(pools, before):
            x.copy_(y)
        fed.copy_(t), m.uniform.copy_(u), m.tokens.fill_(-5)
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip([m.tokens, m.adjusted] + list(pools), w):
            assert torch.equal(x, y)
    assert tle.device_error() == 0
