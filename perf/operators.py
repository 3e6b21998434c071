"""Operators of a serving step over the paged KV cache, as measured cases.

Three operators, each in a plain form (elementary torch operations) and as the
framework's calls:

* ``append``: rope on the q and k of a batch of token chunks, k and v written
  to their rows of the paged cache, q returned rotated
  (``tle.PagedChunkBatch.append``).
* ``attend``: causal attention of those chunks over the paged cache, one token
  per sequence (decode) to whole prompts (``tle.PagedChunkBatch.attend``).
* ``logits``: repetition, frequency and presence penalties, biases and the mask
  of allowed tokens, before a token is sampled (``tle.logits_adjust``).

The rotation is the framework's: pair (2i, 2i+1) of a head turned by the angle
fl32(pos * f_i), f_i = fl32(1 / fl32(base^(2i/64))), the product rounded to 32
bits as its decode rounds it, so that rows written by either call belong to
one cache.
"""
import os
import sys

import numpy as np
import torch

own = False

HD = 64            # width of a head
BASE = 10000.0     # rope base
ALLOWED = 0.3      # share of the vocabulary that a mask lets through


def _tle():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyllama-engine_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tle
    return tle


def _chunks(name, op, **kw):
    c = {"name": name, "op": op, "seqs": 1, "new": 1, "ctx": 0, "ragged": False, "heads": 32, "kv_heads": 4,
         "page": 256, "act": "f32", "pool": "bf16", "layers": 2}
    c.update(kw)
    return c


def _rows(name, **kw):
    c = {"name": name, "op": "logits", "rows": 1, "vocab": 32000, "history": 512, "penalties": True, "biases": 0,
         "mask": False}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of a batch: one new row per sequence, latency counts
        _chunks("append 64x1", "append", seqs=64, new=1, ctx=2047, ragged=True),
        # a whole prompt of the framework's n_ctx into an fp32 cache
        _chunks("append 1x2048 f32", "append", new=2048, pool="f32"),
        # pieces of several prompts, activations in bf16, a small model's heads, odd lengths
        _chunks("append 24x1021 bf16", "append", seqs=24, new=1021, ctx=3001, ragged=True, act="bf16", heads=16, kv_heads=8, page=64),
        # a few guessed tokens checked at once behind one user's context: the smallest call
        _chunks("attend 1x5 at 700", "attend", new=5, ctx=700),
        # one decode step of 64 sequences of 1024 to 2048 rows
        _chunks("attend 64x1 at 2047", "attend", seqs=64, new=1, ctx=2047, ragged=True),
        # pieces of several prompts, each behind its own context
        _chunks("attend 6x509 at 1999 bf16", "attend", seqs=6, new=509, ctx=1999, ragged=True, act="bf16", page=64),
        # a whole prompt of the framework's n_ctx
        _chunks("attend 1x2048 bf16", "attend", new=2048, act="bf16"),
        # a piece of a long prompt, activations in fp32 as the framework's products leave them
        _chunks("attend 1x777 at 16000", "attend", new=777, ctx=16000, page=128),
        # a large piece late in a long prompt: the largest call
        _chunks("attend 1x2048 at 30000 bf16", "attend", new=2048, ctx=30000, act="bf16"),
        # one user's next token: the smallest call
        _rows("logits 1x32000", history=700),
        # a batch's next tokens under a grammar, with biases
        _rows("logits 64x32000 mask", rows=64, history=2048, biases=100, mask=True),
        # a large batch over a larger, odd vocabulary
        _rows("logits 256x100003 mask", rows=256, vocab=100003, history=4001, biases=300, mask=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logits"])
    if op == "logits":
        rows = _log_int(rng, 1, 256)
        c = _rows("", rows=rows, vocab=_log_int(rng, 1000, 100003), history=_log_int(rng, 1, 4001), penalties=rng.random() < 0.8,
                  biases=rng.choice([0, 1, 17, 300]), mask=rng.random() < 0.5)
        del c["name"]
        return c
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (32, 8), (16, 8), (8, 8), (12, 4), (20, 4)])
    act = rng.choice(["f32", "bf16"])
    c = _chunks("", op, heads=heads, kv_heads=kv_heads, act=act, page=rng.choice([64, 128, 256, 1024]), ragged=rng.random() < 0.7)
    del c["name"]
    if op == "append":
        c["seqs"] = _log_int(rng, 1, 64)
        c["new"] = _log_int(rng, 1, max(1, 24000 // c["seqs"] // 2))
        c["ctx"] = rng.choice([0, _log_int(rng, 1, 4096)])
        c["pool"] = rng.choice(["f32", "bf16"])
        return c
    c["seqs"] = _log_int(rng, 1, 64)
    c["new"] = _log_int(rng, 1, max(1, 2048 // c["seqs"]))
    c["ctx"] = rng.choice([0, _log_int(rng, 1, max(2, 60000 // c["seqs"])), _log_int(rng, 1, max(2, 60000 // c["seqs"]))])
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


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, g, dev)
    pos, new = _lengths(case)
    H, KH, page, T = case["heads"], case["kv_heads"], case["page"], sum(new)
    act = torch.float32 if case["act"] == "f32" else torch.bfloat16
    pool = torch.float32 if case["pool"] == "f32" else torch.bfloat16
    need = [-(-(p + m) // page) for p, m in zip(pos, new)]
    n_pages = sum(need) + 3                                # a few pages that no sequence has
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    most = max(need)
    table = torch.zeros(len(pos), most, dtype=torch.int32, device=dev)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = ids[at:at + k]
        at += k
    dims = (case["layers"], n_pages, page, KH * HD)
    st = {"case": case, "layer": case["layers"] - 1, "table": table,
          "pos": torch.tensor(pos, dtype=torch.int32, device=dev),
          "new": torch.tensor(new, dtype=torch.int32, device=dev),
          "most_new": max(new), "tokens": T,
          "q": torch.randn(T, H * HD, generator=g, device=dev).to(act),
          "k": torch.randn(T, KH * HD, generator=g, device=dev).to(act),
          "v": torch.randn(T, KH * HD, generator=g, device=dev).to(act),
          "k_pool": torch.randn(dims, generator=g, device=dev).to(pool),
          "v_pool": torch.randn(dims, generator=g, device=dev).to(pool),
          "out": torch.zeros(T, H * HD, dtype=act, device=dev)}
    if own:
        # what a serving loop keeps: the cache, and the batch of this step with its plan
        tle = _tle()
        cache = tle.PagedKVCache(n_pages, page, tle.Shape(case["layers"], H, KH, HD, BASE), dtype=pool,
                                 pools=(st["k_pool"], st["v_pool"]))
        st["batch"] = tle.PagedChunkBatch(cache, [table[s, :k] for s, k in enumerate(need)], pos, new)
    return st


def _prepare_logits(case, g, dev):
    n, V = case["rows"], case["vocab"]
    r = np.random.RandomState(int(torch.randint(0, 1 << 30, (1,), generator=g, device=dev).item()))
    counts = r.randint((case["history"] + 1) // 2, case["history"] + 1, n)
    start = np.concatenate([[0], np.cumsum(counts)])
    # most of a text's tokens are few common ones
    tokens = np.minimum((V * r.random_sample(start[-1]) ** 4).astype(np.int64), V - 1)
    t = lambda a, d: torch.from_numpy(np.ascontiguousarray(a)).to(dev, d)  # noqa: E731
    st = {"case": case, "logits": 3.0 * torch.randn(n, V, generator=g, device=dev), "out": torch.zeros(n, V, device=dev),
          "tokens": t(tokens, torch.int32), "token_start": t(start, torch.int32), "n_prompt": t(counts // 3, torch.int32),
          "repetition": t(1.0 + 0.5 * r.random_sample(n), torch.float32),
          "frequency": t(0.5 * r.random_sample(n), torch.float32),
          "presence": t(r.random_sample(n), torch.float32)}
    if case["biases"]:
        b = np.full(n, case["biases"])
        st["bias_start"] = t(np.concatenate([[0], np.cumsum(b)]), torch.int32)
        st["bias_tokens"] = t(r.randint(0, V, int(b.sum())), torch.int32)
        st["bias_values"] = t(4.0 * r.standard_normal(int(b.sum())), torch.float32)
    if case["mask"]:
        bits = torch.rand(n, -(-V // 32) * 32, generator=g, device=dev) < ALLOWED
        w = bits.view(n, -1, 32).to(torch.int64) << torch.arange(32, device=dev)
        st["allowed"] = w.sum(-1).to(torch.int32)         # bit t % 32 of word t / 32: token t is allowed
    if own:
        tle = _tle()
        st["rules"] = tle.LogitRules(n, V, **{k: st[k] for k in _given(case)})
    return st


def _given(case):
    keys = []
    if case["penalties"]:
        keys += ["tokens", "token_start", "n_prompt", "repetition", "frequency", "presence"]
    if case["biases"]:
        keys += ["bias_tokens", "bias_values", "bias_start"]
    if case["mask"]:
        keys += ["allowed"]
    return keys


# ---------------------------------------------------------------------- run
def run(st):
    op = st["case"]["op"]
    if own:
        if op == "append":
            st["batch"].append(st["q"], st["k"], st["v"], st["layer"], q_out=st["out"])
            return {"q": st["out"], "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
        if op == "attend":
            st["batch"].attend(st["q"], st["out"], st["layer"])
            return st["out"]
        _tle().logits_adjust(st["out"], st["logits"], st["rules"])
        return st["out"]
    if op == "append":
        return _plain_append(st)
    if op == "attend":
        return _plain_attend(st)
    return _plain_logits(st)


def _token_of(st):
    """For each token: its sequence, and its place in the sequence's chunk."""
    new = st["new"].long()
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=new.device), new, output_size=st["tokens"])
    first = torch.cumsum(new, 0) - new
    return seq, torch.arange(st["tokens"], device=new.device) - first[seq]


def _turn(x, cos, sin):
    y = x.float().view(x.shape[0], -1, HD // 2, 2)
    a, b = y[..., 0], y[..., 1]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).view(x.shape).to(x.dtype)


def _plain_append(st):
    c = st["case"]
    seq, i = _token_of(st)
    p = st["pos"].long()[seq] + i
    two_i = torch.arange(0, HD, 2, device=p.device, dtype=torch.float64)
    freq = 1.0 / torch.pow(BASE, two_i / HD).float()       # both steps rounded to 32 bits, as the framework's table is
    angle = (p.float()[:, None] * freq).double()           # the product in 32 bits, its sine and cosine in 64
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    page = st["table"].long()[seq, p // c["page"]]
    row = p % c["page"]
    kp, vp = st["k_pool"][st["layer"]], st["v_pool"][st["layer"]]
    kp[page, row] = _turn(st["k"].float(), cos, sin).to(kp.dtype)
    vp[page, row] = st["v"].to(vp.dtype)
    st["out"].copy_(_turn(st["q"], cos, sin))
    return {"q": st["out"], "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _plain_attend(st):
    """All sequences at once, padded to the longest chunk and the longest context."""
    c = st["case"]
    H, KH, G = c["heads"], c["kv_heads"], c["heads"] // c["kv_heads"]
    n = c["seqs"]
    seq, i = _token_of(st)
    S = st["most_new"]
    table = st["table"].long()
    R = table.shape[1] * c["page"]
    K = st["k_pool"][st["layer"]][table].view(n, R, KH, HD).float().transpose(1, 2)     # [n, KH, R, HD]
    V = st["v_pool"][st["layer"]][table].view(n, R, KH, HD).float().transpose(1, 2)
    Q = torch.zeros(n, S, H * HD, device=K.device)
    Q[seq, i] = st["q"].float()
    Q = Q.view(n, S, KH, G, HD).permute(0, 2, 3, 1, 4).reshape(n, KH, G * S, HD)        # [n, KH, G*S, HD]
    s = torch.matmul(Q, K.transpose(2, 3)) * (HD ** -0.5)
    last = st["pos"][:, None] + torch.arange(S, device=K.device)                        # [n, S]
    seen = torch.arange(R, device=K.device) <= last[:, :, None]                         # [n, S, R]
    s = s.view(n, KH, G, S, R).masked_fill_(~seen[:, None, None], float("-inf"))
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, KH, G * S, R), V)
    o = o.view(n, KH, G, S, HD).permute(0, 3, 1, 2, 4).reshape(n, S, H * HD)
    return o[seq, i].to(st["q"].dtype)


def _plain_logits(st):
    c = st["case"]
    x = st["logits"]
    n, V = x.shape
    if c["penalties"]:
        start = st["token_start"].long()
        count = start[1:] - start[:-1]
        row = torch.repeat_interleave(torch.arange(n, device=x.device), count, output_size=st["tokens"].numel())
        place = torch.arange(st["tokens"].numel(), device=x.device) - start[row]
        made = (place >= st["n_prompt"].long()[row]).float()
        at = row * V + st["tokens"].long()
        seen = torch.zeros(n * V, device=x.device).index_fill_(0, at, 1.0).view(n, V) > 0
        times = torch.zeros(n * V, device=x.device).index_add_(0, at, made).view(n, V)
        rep = st["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - st["frequency"][:, None] * times - st["presence"][:, None] * (times > 0)
    if c["biases"]:
        start = st["bias_start"].long()
        row = torch.repeat_interleave(torch.arange(n, device=x.device), start[1:] - start[:-1], output_size=st["bias_tokens"].numel())
        x = x + torch.zeros(n * V, device=x.device).index_add_(0, row * V + st["bias_tokens"].long(), st["bias_values"]).view(n, V)
    if c["mask"]:
        bits = (st["allowed"][:, :, None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.view(n, -1)[:, :V] > 0, x, float("-inf"))
    return x if x is not st["logits"] else x.clone()


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "logits":
        n, V = case["rows"], case["vocab"]
        b = 8 * n * V
        if case["penalties"]:
            b += 3 * n * case["history"]                   # three quarters of the longest history on average, 4 bytes each
        b += 8 * n * case["biases"]
        b += n * V // 8 if case["mask"] else 0
        return {"bytes": b, "flops": 4 * n * V}
    pos, new = _lengths(case)
    H, KH = case["heads"], case["kv_heads"]
    a, p = (4 if case["act"] == "f32" else 2), (4 if case["pool"] == "f32" else 2)
    T = sum(new)
    if case["op"] == "append":
        return {"bytes": T * HD * (2 * H * a + 2 * KH * (a + p)), "flops": 3 * T * HD * (H + KH)}
    rows = sum(x + y for x, y in zip(pos, new))
    pairs = sum(y * x + y * (y + 1) // 2 for x, y in zip(pos, new))
    return {"bytes": rows * 2 * KH * HD * p + 2 * T * H * HD * a, "flops": 4 * HD * H * pairs}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "logits":
        return _exact_logits(case, st)
    pos, new = _lengths(case)
    page, KH, layer = case["page"], case["kv_heads"], st["layer"]
    G = case["heads"] // KH
    table = st["table"].cpu().numpy()
    if case["op"] == "append":
        # the angle is a number of 32 bits by definition; everything else is in 64
        freq = np.float32(1) / np.power(np.float64(BASE), np.arange(0, HD, 2) / HD).astype(np.float32)
        where = np.concatenate([np.arange(p, p + m) for p, m in zip(pos, new)])
        angle = (where.astype(np.float32)[:, None] * freq.astype(np.float32)).astype(np.float64)
        z = torch.from_numpy(np.cos(angle) + 1j * np.sin(angle)).to(st["q"].device)

        def turned(x):
            w = torch.view_as_complex(x.double().view(x.shape[0], -1, HD // 2, 2).contiguous()) * z[:, None, :]
            return torch.view_as_real(w).reshape(x.shape)
        flat = np.concatenate([table[s][np.arange(p, p + m) // page].astype(np.int64) * page + np.arange(p, p + m) % page
                               for s, (p, m) in enumerate(zip(pos, new))])
        flat = torch.from_numpy(flat).to(st["q"].device)
        kp, vp = st["k_pool"].double(), st["v_pool"].double()
        kp[layer].view(-1, KH * HD).index_copy_(0, flat, turned(st["k"]))
        vp[layer].view(-1, KH * HD).index_copy_(0, flat, st["v"].double())
        return {"q": turned(st["q"]), "k_pool": kp, "v_pool": vp}
    out = torch.empty(st["tokens"], case["heads"] * HD, dtype=torch.float64, device=st["q"].device)
    t0 = 0
    for s, (p, m) in enumerate(zip(pos, new)):
        ids = torch.from_numpy(table[s].astype(np.int64)).to(out.device)
        hidden = torch.triu(torch.ones(m, p + m, dtype=torch.bool, device=out.device), diagonal=p + 1)
        for h in range(KH):
            k = st["k_pool"][layer, ids, :, h * HD:(h + 1) * HD].reshape(-1, HD)[:p + m].double()
            v = st["v_pool"][layer, ids, :, h * HD:(h + 1) * HD].reshape(-1, HD)[:p + m].double()
            for j in range(h * G, (h + 1) * G):
                e = st["q"][t0:t0 + m, j * HD:(j + 1) * HD].double() @ k.T / 8.0
                e[hidden] = -np.inf
                out[t0:t0 + m, j * HD:(j + 1) * HD] = torch.softmax(e, 1) @ v
        t0 += m
    return out


def _exact_logits(case, st):
    a = {k: v.cpu().numpy() for k, v in st.items() if isinstance(v, torch.Tensor)}
    x = a["logits"].astype(np.float64)
    V = case["vocab"]
    for r in range(case["rows"]):
        y = x[r]
        if case["penalties"]:
            lo, hi, cut = a["token_start"][r], a["token_start"][r + 1], a["n_prompt"][r]
            ids = a["tokens"][lo:hi]
            used = np.unique(ids)
            rep = float(a["repetition"][r])
            y[used] = np.where(y[used] > 0, y[used] / rep, y[used] * rep)
            made, times = np.unique(ids[cut:], return_counts=True)
            y[made] -= float(a["frequency"][r]) * times + float(a["presence"][r])
        if case["biases"]:
            lo, hi = a["bias_start"][r], a["bias_start"][r + 1]
            np.add.at(y, a["bias_tokens"][lo:hi], a["bias_values"][lo:hi].astype(np.float64))
        if case["mask"]:
            bits = np.unpackbits(a["allowed"][r].view(np.uint8), bitorder="little")[:V]
            y[bits == 0] = -np.inf
    return torch.from_numpy(x)
