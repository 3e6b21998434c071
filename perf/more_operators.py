"""Operators of a serving step over a paged KV cache in 8 bits, as measured cases.

Five operators, each in a plain form (elementary torch operations) and as the
framework's calls:

* ``append``: rope by rules (interleaved or half layout, a part of the head,
  given frequencies, a factor on sine and cosine) and RMS norms of the q and k
  heads, for chunks of new tokens; k and v to their rows of fp32 or bf16 pages
  (``tle.PagedChunkBatch.append`` with ``tle.AppendRules``).
* ``store``: the same into pages of 8 bits, and the values read back that the
  new rows now stand for (``append``, then ``read`` of the new rows).
* ``read``: all rows of the sequences of an 8-bit cache, as numbers
  (``tle.PagedChunkBatch.read``).
* ``attend``: causal attention of new tokens over an 8-bit cache
  (``tle.PagedChunkBatch.attend``).
* ``sample``: temperature, top-k, top-p and min-p for a batch of logits, with
  given uniform numbers (``tle.sample_rows``).

The 8-bit form of a head's row x[0..63]: a byte b and 64 whole numbers c in
-127..127 that stand for c * 2^(b - 127), with 2^(b - 127) the smallest power
of two for which no |x| / 2^(b - 127) is above 127, and c the nearest whole
number (ties to even).  So a stored value is a bf16 number exactly.  The pools
are [layers][pages][kv_heads][page rows][64] and [layers][pages][kv_heads][page rows].

The rotation's angle is the number fl32(pos * f_i), as in the framework's other
calls, with the frequencies f_i given.

Sampling: tokens are ranked by their logits (ties: the lower index first), and
weigh exp((x - max) / temperature).  Kept are the first top_k tokens, of these
the ones with a weight of at least min_p times the largest, and of these the
first ones until their weights reach top_p of the sum.  The token is the first
in index order at which the running sum of the kept weights exceeds the uniform
number times their sum.  A temperature of 0 takes the largest logit.
"""
import os
import sys

import numpy as np
import torch

own = False

HD = 64            # width of a head
BASE = 10000.0     # rope base


def _tle():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyllama-engine_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tle
    return tle


def _chunks(name, op, **kw):
    c = {"name": name, "op": op, "seqs": 1, "new": 1, "ctx": 0, "ragged": False, "heads": 32, "kv_heads": 4,
         "page": 256, "act": "f32", "layers": 2}
    if op in ("append", "store"):
        c.update({"layout": "half", "rotary": 64, "stretch": 1.0, "norms": True})
    if op == "append":
        c["pool"] = "bf16"
    c.update(kw)
    return c


def _rows(name, **kw):
    c = {"name": name, "op": "sample", "rows": 1, "vocab": 32000, "top_k": False, "top_p": True, "min_p": False,
         "hidden": 0.0}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of a batch whose q and k heads are normed: latency counts
        _chunks("append 32x1 norms", "append", seqs=32, new=1, ctx=4000, ragged=True),
        # a prompt of twice the framework's n_ctx, its positions scaled, half of each head rotated
        _chunks("append 1x4096 part bf16", "append", new=4096, act="bf16", layout="interleaved", rotary=32, stretch=2.0, norms=False),
        # one decode step into an 8-bit cache: the smallest store
        _chunks("store 48x1", "store", seqs=48, new=1, ctx=2047, ragged=True, norms=False, layout="interleaved"),
        # pieces of several prompts into an 8-bit cache, a small model's heads, odd lengths
        _chunks("store 16x1501 norms bf16", "store", seqs=16, new=1501, ctx=1001, ragged=True, act="bf16", heads=16, kv_heads=8, page=64),
        # one user's cache read back, to be moved elsewhere
        _chunks("read 1 of 700", "read", new=1, ctx=699),
        # a batch's long caches read back
        _chunks("read 24 of 8000 bf16", "read", seqs=24, new=1, ctx=8000, ragged=True, act="bf16", page=128),
        # a few guessed tokens checked at once behind one user's context: the smallest attention
        _chunks("attend 1x4 at 700", "attend", new=4, ctx=700),
        # one decode step of 64 sequences of 1024 to 2048 rows
        _chunks("attend 64x1 at 2047", "attend", seqs=64, new=1, ctx=2047, ragged=True),
        # one decode step of long sequences: the most rows
        _chunks("attend 32x1 at 16000 bf16", "attend", seqs=32, new=1, ctx=16000, ragged=True, act="bf16", page=128),
        # pieces of several prompts, each behind its own context
        _chunks("attend 4x601 at 2999 bf16", "attend", seqs=4, new=601, ctx=2999, ragged=True, act="bf16", page=64),
        # one user's next token: the smallest sampling
        _rows("sample 1x32000", top_k=True),
        # a large batch over a larger, odd vocabulary, some of it masked
        _rows("sample 256x100003", rows=256, vocab=100003, min_p=True, top_k=True, hidden=0.5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "store", "read", "attend", "attend", "attend", "sample", "sample"])
    if op == "sample":
        c = _rows("", rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 1000, 100003), top_k=rng.random() < 0.5,
                  top_p=rng.random() < 0.6, min_p=rng.random() < 0.4, hidden=rng.choice([0.0, 0.0, 0.5, 0.97]))
        del c["name"]
        return c
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (32, 8), (16, 8), (8, 8), (12, 4), (20, 4)])
    c = _chunks("", op, heads=heads, kv_heads=kv_heads, act=rng.choice(["f32", "bf16"]), page=rng.choice([64, 128, 256, 1024]),
                ragged=rng.random() < 0.7)
    del c["name"]
    c["seqs"] = _log_int(rng, 1, 64)
    if op in ("append", "store"):
        c["new"] = _log_int(rng, 1, max(1, 12000 // c["seqs"]))
        c["ctx"] = rng.choice([0, _log_int(rng, 1, 4096)])
        c["layout"] = rng.choice(["half", "interleaved"])
        c["rotary"] = rng.choice([16, 32, 48, 64, 64])
        c["stretch"] = rng.choice([1.0, 2.0, 4.0])
        c["norms"] = rng.random() < 0.6
        if op == "append":
            c["pool"] = rng.choice(["f32", "bf16"])
        return c
    if op == "read":
        c["ctx"] = _log_int(rng, 1, max(2, 120000 // c["seqs"]))
        return c
    c["new"] = 1 if rng.random() < 0.5 else _log_int(rng, 1, max(1, 1200 // c["seqs"]))
    most = 300000 if c["new"] * heads // kv_heads <= 32 else 9000
    c["ctx"] = rng.choice([0, _log_int(rng, 1, max(2, most // c["seqs"])), _log_int(rng, 1, max(2, most // c["seqs"]))])
    c["ctx"] = min(c["ctx"], 30000)
    return c


# ------------------------------------------------------------------- inputs
def _lengths(case):
    """(pos, new) of each sequence: the rows that are in the cache before the
    call and the tokens of its chunk; a ragged batch has half to all of each."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    r = np.random.RandomState(n * 7919 + new * 31 + ctx)
    if not case["ragged"]:
        return [ctx] * n, [new] * n
    return [int(x) for x in r.randint(ctx // 2, ctx + 1, n)], [int(x) for x in r.randint((new + 1) // 2, new + 1, n)]


def _frequencies(rotary, stretch):
    """The frequencies of the rotated pairs, positions stretched where a pair
    turns less than once within 2048 rows, and the factor on sine and cosine."""
    f = BASE ** (-np.arange(0, rotary, 2) / rotary)
    f = np.where(f * 2048 < 2 * np.pi, f / stretch, f)
    return f.astype(np.float32), float(np.float32(1.0 + 0.1 * np.log(stretch)))


def _dtype(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(case, g, dev)
    pos, new = _lengths(case)
    H, KH, page, T, L = case["heads"], case["kv_heads"], case["page"], sum(new), case["layers"]
    act = _dtype(case["act"])
    need = [-(-(p + m) // page) for p, m in zip(pos, new)]
    n_pages = sum(need) + 3                                # a few pages that no sequence has
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(pos), max(need), dtype=torch.int32, device=dev)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = ids[at:at + k]
        at += k
    st = {"case": case, "layer": L - 1, "table": table, "tokens": T, "rows": sum(pos) + T, "most_new": max(new),
          "most_rows": max(p + m for p, m in zip(pos, new)),
          "pos": torch.tensor(pos, dtype=torch.int32, device=dev), "new": torch.tensor(new, dtype=torch.int32, device=dev)}
    rnd = lambda *dims: torch.randn(dims, generator=g, device=dev)  # noqa: E731
    if case["op"] == "append":
        dims = (L, n_pages, page, KH * HD)
        st["k_pool"], st["v_pool"] = rnd(*dims).to(_dtype(case["pool"])), rnd(*dims).to(_dtype(case["pool"]))
    else:
        dims = (L, n_pages, KH, page)
        # rows of different sizes: a tenth of them eight times the others'
        size = lambda: 1.0 + 7.0 * (torch.rand(dims + (1,), generator=g, device=dev) < 0.1)  # noqa: E731
        st["k_codes"], st["k_scale"] = _to_8_bits(rnd(*dims, HD))
        st["v_codes"], st["v_scale"] = _to_8_bits(rnd(*dims, HD) * size())
    if case["op"] != "read":
        st["q"] = rnd(T, H * HD).to(act)
        st["out"] = torch.zeros(T, H * HD, dtype=act, device=dev)
    if case["op"] in ("append", "store"):
        st["k"], st["v"] = rnd(T, KH * HD).to(act), rnd(T, KH * HD).to(act)
        st["freq"], st["factor"] = _frequencies(case["rotary"], case["stretch"])
        if case["norms"]:
            st["q_norm"], st["k_norm"] = 1.0 + 0.2 * rnd(HD), 1.0 + 0.2 * rnd(HD)
    if case["op"] in ("read", "store"):
        n, t = (T, torch.bfloat16) if case["op"] == "store" else (st["rows"], act)
        st["k_out"], st["v_out"] = (torch.zeros(n, KH * HD, dtype=t, device=dev) for _ in range(2))
    if own:
        # what a serving loop keeps: the cache, the batch of this step with its plan, the model's rules
        tle = _tle()
        bits8 = "k_codes" in st
        pools = tuple(st[k] for k in (("k_codes", "v_codes", "k_scale", "v_scale") if bits8 else ("k_pool", "v_pool")))
        cache = tle.PagedKVCache(n_pages, page, tle.Shape(L, H, KH, HD, BASE), dtype=pools[0].dtype, pools=pools)
        st["batch"] = tle.PagedChunkBatch(cache, [table[s, :k] for s, k in enumerate(need)], pos, new)
        if "freq" in st:
            st["rules"] = tle.AppendRules(layout=case["layout"], inv_freq=st["freq"], rope_factor=st["factor"],
                                          q_norm=st.get("q_norm"), k_norm=st.get("k_norm"), eps=1e-5)
    return st


def _power32(e):
    """2^e of whole numbers -126 <= e <= 127, in 32 bits and exact (many rows have numbers half-way between two codes)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _power64(e):
    """2^e of whole numbers, in 64 bits and exact."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _to_8_bits(x):
    """Whole numbers (int8) and the byte of the power of two (uint8) of rows of finite numbers."""
    most = x.abs().amax(-1)
    # 127 * 2^e as a number of 32 bits is exact, so that the comparison is
    e = torch.frexp(most)[1] - 7                           # most < 2^(e + 7): e or e + 1
    e = torch.where(most > 127.0 * _power32(e), e + 1, e).clamp_(min=-126)
    codes = torch.round(x * _power32(-e)[..., None])
    return codes.to(torch.int8), (e + 127).to(torch.uint8)


def _from_8_bits(codes, scale):
    return codes.float() * _power32(scale.int() - 127)[..., None]


def _prepare_sample(case, g, dev):
    n, V = case["rows"], case["vocab"]
    r = np.random.RandomState(int(torch.randint(0, 1 << 30, (1,), generator=g, device=dev).item()))
    x = 2.0 * torch.randn(n, V, generator=g, device=dev)
    # a few likely tokens per row, as after a text: some rows nearly sure, some not
    few = torch.randint(0, V, (n, 24), generator=g, device=dev)
    x.scatter_add_(1, few, 10.0 * torch.rand(n, 24, generator=g, device=dev) * torch.rand(n, 1, generator=g, device=dev))
    if case["hidden"]:
        x.masked_fill_(torch.rand(n, V, generator=g, device=dev) < case["hidden"], float("-inf"))
    t = lambda a, d: torch.from_numpy(np.ascontiguousarray(a)).to(dev, d)  # noqa: E731
    temperature = r.uniform(0.5, 1.3, n)
    temperature[r.random_sample(n) < 0.1] = 0.0            # some requests are greedy
    st = {"case": case, "logits": x, "out": torch.zeros(n, dtype=torch.int32, device=dev),
          "uniform": torch.rand(n, generator=g, device=dev), "temperature": t(temperature, torch.float32)}
    if case["top_k"]:
        st["top_k"] = t(np.where(r.random_sample(n) < 0.3, 0, (2000.0 ** r.random_sample(n)).astype(np.int64)), torch.int32)
    if case["top_p"]:
        st["top_p"] = t(np.where(r.random_sample(n) < 0.2, 1.0, r.uniform(0.5, 0.99, n)), torch.float32)
    if case["min_p"]:
        st["min_p"] = t(np.where(r.random_sample(n) < 0.3, 0.0, r.uniform(0.001, 0.2, n)), torch.float32)
    if own:
        tle = _tle()
        st["rules"] = tle.SampleRules(n, V, **{k: st[k] for k in ("temperature", "top_k", "top_p", "min_p") if k in st})
    return st


# ---------------------------------------------------------------------- run
def run(st):
    op = st["case"]["op"]
    if own:
        if op == "sample":
            _tle().sample_rows(st["out"], st["logits"], st["rules"], st["uniform"])
            return st["out"]
        if op == "attend":
            st["batch"].attend(st["q"], st["out"], st["layer"])
            return st["out"]
        if op == "read":
            st["batch"].read(st["k_out"], st["v_out"], st["layer"])
            return {"k": st["k_out"], "v": st["v_out"]}
        st["batch"].append(st["q"], st["k"], st["v"], st["layer"], q_out=st["out"], rules=st["rules"])
        if op == "append":
            return {"q": st["out"], "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
        st["batch"].read(st["k_out"], st["v_out"], st["layer"], new_only=True)
        return {"q": st["out"], "k": st["k_out"], "v": st["v_out"]}
    return {"append": _plain_append, "store": _plain_append, "read": _plain_read, "attend": _plain_attend,
            "sample": _plain_sample}[op](st)


def _place(count, total):
    """For `total` things of sequences with `count` each: the sequence, and the place in it."""
    count = count.long()
    seq = torch.repeat_interleave(torch.arange(count.numel(), device=count.device), count, output_size=total)
    first = torch.cumsum(count, 0) - count
    return seq, torch.arange(total, device=count.device) - first[seq]


def _headed(x, st, cos, sin, norm):
    """Norm and rotation of the heads of x, in 32 bits: [tokens][heads][64]."""
    c = st["case"]
    y = x.float().view(x.shape[0], -1, HD)
    if norm is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * norm
    R = c["rotary"]
    z, rest = y[..., :R], y[..., R:]
    if c["layout"] == "half":
        a, b = z[..., :R // 2], z[..., R // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b = z[..., 0::2], z[..., 1::2]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)


def _plain_append(st):
    c = st["case"]
    seq, i = _place(st["new"], st["tokens"])
    p = st["pos"].long()[seq] + i
    freq = torch.from_numpy(st["freq"]).to(p.device)
    angle = (p.float()[:, None] * freq).double()           # the product in 32 bits, its sine and cosine in 64
    cos, sin = ((f(angle) * st["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    page = st["table"].long()[seq, p // c["page"]]
    row = p % c["page"]
    st["out"].copy_(_headed(st["q"], st, cos, sin, st.get("q_norm")).view(st["out"].shape))
    k = _headed(st["k"], st, cos, sin, st.get("k_norm"))
    v = st["v"].float().view(k.shape)
    if c["op"] == "append":
        kp, vp = st["k_pool"][st["layer"]], st["v_pool"][st["layer"]]
        kp[page, row] = k.flatten(1).to(kp.dtype)
        vp[page, row] = v.flatten(1).to(vp.dtype)
        return {"q": st["out"], "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
    kc, ks = _to_8_bits(k)
    vc, vs = _to_8_bits(v)
    st["k_codes"][st["layer"]][page, :, row] = kc
    st["k_scale"][st["layer"]][page, :, row] = ks
    st["v_codes"][st["layer"]][page, :, row] = vc
    st["v_scale"][st["layer"]][page, :, row] = vs
    st["k_out"].copy_(_from_8_bits(kc, ks).flatten(1))
    st["v_out"].copy_(_from_8_bits(vc, vs).flatten(1))
    return {"q": st["out"], "k": st["k_out"], "v": st["v_out"]}


def _plain_read(st):
    c = st["case"]
    seq, p = _place(st["pos"] + st["new"], st["rows"])
    page = st["table"].long()[seq, p // c["page"]]
    row = p % c["page"]
    for x in "kv":
        codes, scale = st[x + "_codes"][st["layer"]], st[x + "_scale"][st["layer"]]
        st[x + "_out"].copy_(_from_8_bits(codes[page, :, row], scale[page, :, row]).flatten(1))
    return {"k": st["k_out"], "v": st["v_out"]}


def _plain_attend(st):
    """All sequences at once, padded to the longest chunk and the longest context."""
    c = st["case"]
    H, KH, G, n = c["heads"], c["kv_heads"], c["heads"] // c["kv_heads"], c["seqs"]
    seq, i = _place(st["new"], st["tokens"])
    S, R = st["most_new"], st["most_rows"]
    table = st["table"].long()

    def rows(x):                                                                        # [n, KH, R, HD]
        codes, scale = st[x + "_codes"][st["layer"]][table], st[x + "_scale"][st["layer"]][table]
        y = _from_8_bits(codes, scale).transpose(1, 2)
        return y.reshape(n, KH, -1, HD)[:, :, :R]

    Q = torch.zeros(n, S, H * HD, device=table.device)
    Q[seq, i] = st["q"].float()
    Q = Q.view(n, S, KH, G, HD).permute(0, 2, 3, 1, 4).reshape(n, KH, G * S, HD)        # [n, KH, G*S, HD]
    s = torch.matmul(Q, rows("k").transpose(2, 3)) * (HD ** -0.5)
    last = st["pos"][:, None] + torch.arange(S, device=s.device)                        # [n, S]
    seen = torch.arange(R, device=s.device) <= last[:, :, None]                         # [n, S, R]
    s = s.view(n, KH, G, S, R).masked_fill_(~seen[:, None, None], float("-inf"))
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, KH, G * S, R), rows("v"))
    o = o.view(n, KH, G, S, HD).permute(0, 3, 1, 2, 4).reshape(n, S, H * HD)
    st["out"].copy_(o[seq, i])
    return st["out"]


def _plain_sample(st):
    x = st["logits"]
    n, V = x.shape
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    T = st["temperature"].double()[:, None]
    w = torch.exp((xs.double() - xs[:, :1].double()) / torch.where(T > 0, T, 1.0))       # by rank, the largest is 1
    rank = torch.arange(V, device=x.device)
    if "top_k" in st:
        k = st["top_k"][:, None]
        w = torch.where((rank < k) | (k <= 0), w, 0.0)
    if "min_p" in st:
        w = torch.where(w >= st["min_p"].double()[:, None], w, 0.0)
    if "top_p" in st:
        p = st["top_p"].double()[:, None]
        run_ = torch.cumsum(w, 1)
        w = torch.where((run_ - w < p * run_[:, -1:]) | (p >= 1), w, 0.0)
    run_ = torch.cumsum(torch.zeros_like(w).scatter_(1, order, w), 1)                     # in index order
    at = torch.searchsorted(run_, st["uniform"].double()[:, None] * run_[:, -1:], right=True)[:, 0].clamp_(max=V - 1)
    st["out"].copy_(torch.where(T[:, 0] > 0, at, order[:, 0]))
    return st["out"]


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "sample":
        n, V = case["rows"], case["vocab"]
        return {"bytes": 4 * n * V + 24 * n, "flops": 20 * n * V}
    pos, new = _lengths(case)
    H, KH = case["heads"], case["kv_heads"]
    a, T = (4 if case["act"] == "f32" else 2), sum(new)
    rows = sum(pos) + T
    row8 = 2 * KH * (HD + 1)                               # a stored row of K and V
    if case["op"] == "append":
        p = 4 if case["pool"] == "f32" else 2
        return {"bytes": T * HD * (2 * H * a + 2 * KH * (a + p)), "flops": 8 * T * HD * (H + KH)}
    if case["op"] == "store":                              # the stored rows are written, and read again for their values
        return {"bytes": T * (HD * (2 * H * a + 2 * KH * a) + 2 * row8 + 2 * KH * HD * 2), "flops": 10 * T * HD * (H + 2 * KH)}
    if case["op"] == "read":
        return {"bytes": rows * (row8 + 2 * KH * HD * a), "flops": 2 * rows * KH * HD}
    pairs = sum(y * x + y * (y + 1) // 2 for x, y in zip(pos, new))
    return {"bytes": rows * row8 + 2 * T * H * HD * a, "flops": 4 * HD * H * pairs}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "sample":
        return _exact_sample(st)
    pos, new = _lengths(case)
    page, KH, layer = case["page"], case["kv_heads"], st["layer"]
    table = st["table"].cpu().numpy().astype(np.int64)
    dev = st["table"].device

    def flat(s, first, end):
        """Rows of sequence s as rows of a layer's pages, one after another."""
        r = np.arange(first, end)
        return torch.from_numpy(table[s][r // page] * page + r % page).to(dev)

    def stored(x, s, h, end):
        """Head h of sequence s's first rows in the 8-bit pool: [end][64]."""
        at = flat(s, 0, end)
        codes, b = (st[x + y][layer, :, h].reshape(-1, *d)[at] for y, d in (("_codes", (HD,)), ("_scale", ())))
        return codes.double() * _power64(b.long() - 127)[:, None]

    if case["op"] == "read":
        got = {x: torch.cat([torch.cat([stored(x, s, h, p + m) for h in range(KH)], 1) for s, (p, m) in enumerate(zip(pos, new))])
               for x in "kv"}
        return got
    if case["op"] == "attend":
        G = case["heads"] // KH
        out = torch.empty(st["tokens"], case["heads"] * HD, dtype=torch.float64, device=dev)
        t0 = 0
        for s, (p, m) in enumerate(zip(pos, new)):
            hidden = torch.triu(torch.ones(m, p + m, dtype=torch.bool, device=dev), diagonal=p + 1)
            for h in range(KH):
                k, v = stored("k", s, h, p + m), stored("v", s, h, p + m)
                for j in range(h * G, (h + 1) * G):
                    e = st["q"][t0:t0 + m, j * HD:(j + 1) * HD].double() @ k.T / 8.0
                    e[hidden] = -np.inf
                    out[t0:t0 + m, j * HD:(j + 1) * HD] = torch.softmax(e, 1) @ v
            t0 += m
        return out
    # append and store: the angle is a number of 32 bits by definition; everything else is in 64
    R = case["rotary"]
    where = np.concatenate([np.arange(p, p + m) for p, m in zip(pos, new)])
    angle = (where.astype(np.float32)[:, None] * st["freq"]).astype(np.float64)
    z = torch.from_numpy(st["factor"] * (np.cos(angle) + 1j * np.sin(angle))).to(dev)[:, None]
    first, second = (slice(0, R // 2), slice(R // 2, R)) if case["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))

    def headed(x, norm):
        y = x.double().reshape(x.shape[0], -1, HD).clone()
        if norm is not None:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / HD + 1e-5) * norm.double()
        turned = torch.complex(y[..., first], y[..., second]) * z
        y[..., first], y[..., second] = turned.real, turned.imag
        return y

    q, k, v = headed(st["q"], st.get("q_norm")), headed(st["k"], st.get("k_norm")), st["v"].double().view(-1, KH, HD)
    if case["op"] == "append":
        kp, vp = st["k_pool"].double(), st["v_pool"].double()
        at = torch.cat([flat(s, p, p + m) for s, (p, m) in enumerate(zip(pos, new))])
        kp[layer].view(-1, KH * HD).index_copy_(0, at, k.flatten(1))
        vp[layer].view(-1, KH * HD).index_copy_(0, at, v.flatten(1))
        return {"q": q.flatten(1), "k_pool": kp, "v_pool": vp}

    def rounded(x):
        most = x.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(most.clamp(min=2.0 ** -120))).long() - 8     # from below, up to the first that is enough
        for _ in range(4):
            e = torch.where(127 * _power64(e) < most, e + 1, e)
        step = _power64(e.clamp(min=-126))
        return (torch.round(x / step) * step).flatten(1)

    return {"q": q.flatten(1), "k": rounded(k), "v": rounded(v)}


def _exact_sample(st):
    a = {k: v.cpu().numpy() for k, v in st.items() if isinstance(v, torch.Tensor)}
    got = np.empty(len(a["logits"]), np.int32)
    for r, x in enumerate(a["logits"].astype(np.float64)):
        order = np.argsort(-x, kind="stable")
        T = float(a["temperature"][r])
        if T == 0:
            got[r] = order[0]
            continue
        keep = order[:int(a["top_k"][r])] if "top_k" in a and a["top_k"][r] > 0 else order
        w = np.exp((x[keep] - x[order[0]]) / T)
        if "min_p" in a:
            w = w[w >= float(a["min_p"][r])]
        if "top_p" in a and a["top_p"][r] < 1:
            sums = np.cumsum(w)
            w = w[:1 + int(np.searchsorted(sums, float(a["top_p"][r]) * sums[-1]))]
        by_index = np.argsort(keep[:len(w)])
        sums = np.cumsum(w[by_index])
        got[r] = keep[by_index[int(np.searchsorted(sums, float(a["uniform"][r]) * sums[-1], side="right"))]]
    return torch.from_numpy(got)
