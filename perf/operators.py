"""What is measured of the generation operators: appending to the paged 4-bit key/value cache, attention over that
cache, and sampling.

`run` makes the calls of a decoding program where `own` is true, and computes the same in elementary torch
operations where it is false.  `exact` computes them from their definitions in 64 bits.

The cache: a pool of `pages` pages for the keys and one for the values.  Page p holds, for each key/value head h, one
chunk of page * head_dim * 9/16 bytes: the 4-bit codes of its tokens ([page][head_dim/2] bytes, element 2i in the low
half of byte i, element 2i + 1 in the high half), then their scales ([page][head_dim/32] halves).  An element is
scale * (code - 8).
"""
import math

import torch

own = False

GROUP = 32  # elements that share a scale
FIXED = 2.0 ** 42  # a sampling weight is held as a whole number of 2^-42

_ctx = None


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one token each for a few users: the latency of the cache's update in every layer of a decoding step
        dict(name="append-step", op="append", seqs=8, new=1, length=700, spread=0.5, heads=32, kv_heads=4, head_dim=64, page=16, pages=512),
        # a batch of whole prompts enters the cache (the benchmark's decoder at its training batch)
        dict(name="append-prompts", op="append", seqs=4, new=1024, length=1024, spread=0.0, heads=32, kv_heads=4, head_dim=64, page=16, pages=320),
        # prompts of odd lengths behind a longer past, wide heads, pages that are no power of two
        dict(name="append-ragged", op="append", seqs=13, new=1501, length=5003, spread=0.6, heads=32, kv_heads=8, head_dim=128, page=48, pages=1600),
        # the smallest decoding step: one short sequence, few heads
        dict(name="attend-one", op="attend", seqs=1, new=1, length=203, spread=0.0, heads=8, kv_heads=4, head_dim=64, page=16, pages=64),
        # ordinary serving: a batch of one-token steps over sequences of mixed lengths
        dict(name="attend-batch", op="attend", seqs=32, new=1, length=2048, spread=0.7, heads=32, kv_heads=4, head_dim=64, page=16, pages=4200),
        # many users with long histories, wide heads: the largest cache read
        dict(name="attend-large", op="attend", seqs=64, new=1, length=8192, spread=0.5, heads=32, kv_heads=8, head_dim=128, page=64, pages=8400),
        # one user with one very long history: few rows, so the work has to be split along it
        dict(name="attend-long", op="attend", seqs=1, new=1, length=131072, spread=0.0, heads=32, kv_heads=4, head_dim=64, page=64, pages=2200),
        # a few drafted tokens checked at once for each sequence
        dict(name="attend-draft", op="attend", seqs=16, new=5, length=2901, spread=0.5, heads=32, kv_heads=8, head_dim=128, page=32, pages=1600),
        # the next chunk of long prompts: many query rows on a cached past
        dict(name="attend-chunk", op="attend", seqs=4, new=512, length=4096, spread=0.4, heads=32, kv_heads=4, head_dim=64, page=16, pages=1100),
        # one user's next token
        dict(name="sample-one", op="sample", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0, mixed=False),
        # a batch in which every user has settings of their own
        dict(name="sample-batch", op="sample", rows=128, vocab=32000, temperature=1.0, top_k=50, top_p=0.9, min_p=0.05, mixed=True),
        # a wide vocabulary of odd size, nucleus sampling without a top-k: thousands of tokens stay
        dict(name="sample-wide", op="sample", rows=256, vocab=131075, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, mixed=False),
    ]


def _spread_over(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "sample", "sample"])
    if op == "sample":
        vocab = _spread_over(rng, 200, 140000)
        return dict(op=op, rows=_spread_over(rng, 1, max(1, min(300, 30000000 // vocab))), vocab=vocab, temperature=rng.choice([0.3, 0.8, 1.0, 1.5]), top_k=rng.choice([0, 1, 20, 50, 1000]),
                    top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.02, 0.1]), mixed=rng.random() < 0.5)
    head_dim = rng.choice([32, 64, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if op == "append":
        new = rng.choice([1, _spread_over(rng, 2, 1500)])
        length = new + _spread_over(rng, 1, 4000)
        seqs = _spread_over(rng, 1, max(1, min(64, 16000 // new)))
    else:
        new = rng.choice([1, 1, 1, _spread_over(rng, 2, 8), _spread_over(rng, 9, 400)])
        length = new + _spread_over(rng, 1, 60000 if new == 1 else 5000)
        most = 250000 if new == 1 else 4000000 // new // 32
        seqs = _spread_over(rng, 1, max(1, min(64, most // length)))
    need = seqs * -(-length // page)
    return dict(op=op, seqs=seqs, new=new, length=length, spread=rng.choice([0.0, 0.3, 0.7]), heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=need + rng.randint(1, 20))


def _counts(case):
    """(new tokens, tokens in the cache with the new ones) of each sequence: fixed by the case, mixed lengths."""
    news, lens = [], []
    for b in range(case["seqs"]):
        f = (b * 0.6180339887498949) % 1.0
        n = case["new"] if case["new"] < 9 else max(1, int(case["new"] * (1 - case["spread"] * f)))
        news.append(n)
        lens.append(max(n, int(case["length"] * (1 - case["spread"] * f))))
    return news, lens


def work(case):
    if case["op"] == "sample":
        # every logit read once and compared; settings, token and log-probability
        return {"bytes": case["rows"] * (4 * case["vocab"] + 32), "flops": 2 * case["rows"] * case["vocab"]}
    news, lens = _counts(case)
    H, Hkv, hd, T = case["heads"], case["kv_heads"], case["head_dim"], sum(news)
    held = 2 * Hkv * hd * 9 / 16  # bytes of one token in the cache
    if case["op"] == "append":
        # q, k, v read, q rotated, the codes written; then the new tokens read back as numbers
        moved = T * ((H + 2 * Hkv) * hd * 4 + H * hd * 4 + held) + T * (held + 2 * Hkv * hd * 4)
        return {"bytes": moved + max(lens) * hd * 4, "flops": 3 * T * (H + 2 * Hkv) * hd}
    pairs = sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(news, lens))
    return {"bytes": sum(lens) * held + T * H * (8 * hd + 4), "flops": 4 * pairs * H * hd}


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        logits = normal(R, V) * 2.5
        logits[:, :: 97] += 3.0  # a few likely tokens, as a trained model gives them
        temperature = torch.full((R,), case["temperature"], device="cuda")
        top_k = torch.full((R,), case["top_k"], dtype=torch.int32, device="cuda")
        top_p = torch.full((R,), case["top_p"], device="cuda")
        min_p = torch.full((R,), case["min_p"], device="cuda")
        if case["mixed"]:  # every fourth row greedy, without a top-k, without a nucleus, or all of the case's settings
            i = torch.arange(R, device="cuda") % 4
            temperature[i == 0] = 0.0
            top_k[i == 1] = 0
            top_p[i == 2] = 1.0
            min_p[i == 3] = 0.0
        return dict(op="sample", logits=logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, uniform=torch.rand(R, device="cuda", generator=g),
                    tokens=torch.empty(R, dtype=torch.int64, device="cuda"), logp=torch.empty(R, device="cuda"))

    news, lens = _counts(case)
    H, Hkv, hd, page, pages, T = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["pages"], sum(news)
    width = max(-(-n // page) for n in lens)
    s = dict(op=case["op"], heads=H, kv_heads=Hkv, head_dim=hd, page=page, pages=pages, most=max(news))
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if max(news) > 1 else None
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # row t is token `row_at[t]` of sequence `row_seq[t]`: what a program that batches them knows
    per = torch.tensor(news, device="cuda")
    s["row_seq"] = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), per)
    s["row_at"] = torch.arange(T, device="cuda") - torch.tensor(starts[:-1], device="cuda")[s["row_seq"]] + (torch.tensor(lens, device="cuda") - per)[s["row_seq"]]
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        table[b, :k] = order[at:at + k]
        at += k
    s["table"] = table
    codes, scales = page * hd // 2, page * hd // GROUP
    for name in ("k", "v"):
        pool = torch.empty(pages, Hkv, codes + 2 * scales, dtype=torch.uint8, device="cuda")
        if case["op"] == "attend":
            step = max(1, (1 << 26) // (Hkv * codes))
            for p in range(0, pages, step):
                m = min(step, pages - p)
                # codes and scales as quantised normal values have them: the largest of 32 is about 2.1, either sign
                c = (normal(m, Hkv, codes, 2) * 3.8 + 8).round_().clamp_(0, 15).to(torch.uint8)
                pool[p:p + m, :, :codes] = c[..., 0] | (c[..., 1] << 4)
                d = (2.1 + 0.4 * normal(m, Hkv, scales)) / 8 * torch.sign(normal(m, Hkv, scales))
                pool[p:p + m, :, codes:] = d.half().view(torch.uint8)
        else:
            pool.zero_()
        s[name + "_pool"] = pool
    # q, k and v are columns of one projection's rows
    s["qkv"] = normal(T, (H + 2 * Hkv) * hd) if case["op"] == "append" else normal(T, H * hd) * 2.0
    if case["op"] == "append":
        pos = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None]
        f = 10000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda", dtype=torch.float64) / hd)
        s["cos"], s["sin"] = torch.cos(pos * f).float(), torch.sin(pos * f).float()
        s["q_out"] = torch.empty(T, H * hd, device="cuda")
        s["k_out"], s["v_out"] = torch.empty(T, Hkv * hd, device="cuda"), torch.empty(T, Hkv * hd, device="cuda")
    else:
        s["out"] = torch.empty(T, H * hd, device="cuda")
        s["lse"] = torch.empty(T, H, device="cuda")
    return s


# ------------------------------------------------------------------ the framework's calls


def _framework():
    global _ctx
    if _ctx is None:
        from gollama_b200.device import Context

        _ctx = Context(torch.cuda.current_device())
    return _ctx


def _own_run(s):
    import ctypes as C

    ctx = _framework()
    if s["op"] == "sample":
        R, V = s["logits"].shape
        ctx.call("glc_sample", s["logits"].data_ptr(), V, R, V, s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["uniform"].data_ptr(),
                 s["tokens"].data_ptr(), s["logp"].data_ptr())
        return dict(tokens=s["tokens"], logp=s["logp"])
    if "cache" not in s:  # the handles that a decoding program keeps
        from gollama_b200._lib import KVBatchC, KVCacheC

        s["cache"] = KVCacheC(k=s["k_pool"].data_ptr(), v=s["v_pool"].data_ptr(), num_pages=s["pages"], page_size=s["page"], num_kv_heads=s["kv_heads"], head_dim=s["head_dim"])
        s["batch"] = KVBatchC(page_table=s["table"].data_ptr(), lens=s["lens"].data_ptr(), starts=0 if s["starts"] is None else s["starts"].data_ptr(), num_seqs=s["table"].shape[0],
                              max_pages=s["table"].shape[1], num_rows=s["qkv"].shape[0])
    cache, batch, H = C.byref(s["cache"]), C.byref(s["batch"]), s["heads"]
    qkv, ld, n = s["qkv"].data_ptr(), s["qkv"].shape[1], s["heads"] * s["head_dim"]
    if s["op"] == "append":
        w = s["kv_heads"] * s["head_dim"]
        ctx.call("glc_kv_append", cache, batch, qkv, ld, s["q_out"].data_ptr(), n, H, qkv + 4 * n, ld, qkv + 4 * (n + w), ld, s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0])
        ctx.call("glc_kv_read", cache, batch, s["k_out"].data_ptr(), w, s["v_out"].data_ptr(), w)
        return dict(q=s["q_out"], k=s["k_out"], v=s["v_out"])
    ctx.call("glc_attention_kv", cache, batch, qkv, ld, H, s["out"].data_ptr(), n, s["lse"].data_ptr())
    return dict(out=s["out"], lse=s["lse"])


# ------------------------------------------------------------------ the plain form


def _views(pool, s):
    """The codes [pages, heads, page, head_dim/2] and scales [pages, heads, page, head_dim/32] of a pool."""
    P, h, page, hd = s["pages"], s["kv_heads"], s["page"], s["head_dim"]
    codes = pool[:, :, : page * hd // 2].unflatten(2, (page, hd // 2))
    return codes, pool[:, :, page * hd // 2:].view(torch.float16).unflatten(2, (page, hd // GROUP))


def _numbers(codes, scales):
    """The fp32 numbers [..., head_dim] that codes and scales stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _plain_append(s):
    H, Hkv, hd, page = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, H + 2 * Hkv, hd)
    c, n = s["cos"][s["row_at"]][:, None], s["sin"][s["row_at"]][:, None]
    a, b = x[:, : H + Hkv, 0::2], x[:, : H + Hkv, 1::2]
    turned = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
    where = s["table"][s["row_seq"], s["row_at"] // page].long()
    slot = s["row_at"] % page
    got = dict(q=turned[:, :H].reshape(T, H * hd))
    for name, y in (("k", turned[:, H:]), ("v", x[:, H + Hkv:])):
        y = y.unflatten(-1, (-1, GROUP))
        first = y.abs().argmax(-1, keepdim=True)
        d = (y.gather(-1, first) / -8.0).clamp(-65504, 65504).half()
        q = torch.where(d == 0, 0.0, y.double() / d.double()).round().clamp(-8, 7) + 8
        q = q.to(torch.uint8).flatten(-2)
        codes, scales = _views(s[name + "_pool"], s)
        codes[where, :, slot] = q[..., 0::2] | (q[..., 1::2] << 4)
        scales[where, :, slot] = d[..., 0]
        got[name] = _numbers(codes[where, :, slot], scales[where, :, slot]).reshape(T, Hkv * hd)
    return got


def _plain_attend(s):
    H, Hkv, hd, page = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    G, T, B = H // Hkv, s["qkv"].shape[0], s["table"].shape[0]
    held = []
    for name in ("k", "v"):
        codes, scales = _views(s[name + "_pool"], s)
        t = s["table"].clamp(min=0).long()
        held.append(_numbers(codes[t], scales[t]).transpose(1, 2).flatten(2, 3))  # [B, Hkv, L, hd]
    k, v = held
    # the rows of each sequence, padded to the longest
    if s["starts"] is None:
        at, most = torch.zeros(T, dtype=torch.int64, device=k.device), 1
    else:
        at = torch.arange(T, device=k.device) - s["starts"].long()[s["row_seq"]]
        most = s["most"]
    q = torch.zeros(B, most, H, hd, device=k.device)
    q[s["row_seq"], at] = s["qkv"].view(T, H, hd)
    last = torch.full((B, most), -1, dtype=torch.int64, device=k.device)
    last[s["row_seq"], at] = s["row_at"]
    q = q.view(B, most, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * most, hd)
    scores = (q @ k.transpose(2, 3)).view(B, Hkv, G, most, -1) * (1.0 / math.sqrt(hd))
    seen = torch.arange(k.shape[2], device=k.device) <= last[:, None, None, :, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, G * most, -1) @ v).view(B, Hkv, G, most, hd) / total
    lse = (torch.log(total) + top)[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, H * hd)[s["row_seq"], at]
    return dict(out=o, lse=lse.permute(0, 3, 1, 2).reshape(B, most, H)[s["row_seq"], at])


def _plain_sample(s):
    logits = s["logits"].masked_fill(s["logits"].isnan(), float("-inf"))
    R, V = logits.shape
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    place = torch.arange(V, device=logits.device)
    top = order.values[:, :1].double()
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    e = torch.exp((order.values.double() - top) / torch.where(greedy, 1.0, t))
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k <= 0, V, k))
    e = torch.where(place < k, e, 0.0)
    upto = torch.cumsum(e, 1)
    p = s["top_p"].double()[:, None]
    keep = (place < k) & ((upto - e < p * upto[:, -1:]) | (place == 0) | (p >= 1)) & (e >= s["min_p"].double()[:, None])
    w = torch.zeros_like(e).scatter_(1, order.indices, torch.where(keep, e, 0.0))
    upto = torch.cumsum(w, 1)
    goal = s["uniform"].double()[:, None] * upto[:, -1:]
    token = (upto <= goal).sum(1, keepdim=True).clamp(max=V - 1)
    return dict(tokens=token[:, 0], logp=torch.log(w.gather(1, token) / upto[:, -1:])[:, 0].float())


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[state["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "sample":
        # from the definition, row by row: tokens in falling order, the kept ones' weights, the first whose running
        # sum in vocabulary order passes the goal
        tokens, logp = [], []
        for r in range(case["rows"]):
            x = s["logits"][r].double()
            t, k, p, m, u = (s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
            if not t > 0:
                tokens.append(int(torch.argmax(x)))
                logp.append(0.0)
                continue
            w, idx = torch.sort(torch.exp((x - x.max()) / t), descending=True, stable=True)
            n = case["vocab"] if k <= 0 else min(k, case["vocab"])
            before = torch.cumsum(w[:n], 0) - w[:n]
            n = n if p >= 1 else max(1, int((before < p * w[:n].sum()).sum()))
            n = min(n, max(1, int((w >= m).sum())))
            kept = torch.sort(idx[:n]).values
            w = torch.exp((x[kept] - x.max()) / t)
            run_, all_ = torch.cumsum(w, 0), w.sum()
            j = min(int((run_ <= u * all_).sum()), n - 1)
            tokens.append(int(kept[j]))
            logp.append(float(torch.log(w[j] / all_)))
        return dict(tokens=torch.tensor(tokens), logp=torch.tensor(logp, dtype=torch.float64))
    news, lens = _counts(case)
    H, Hkv, hd, page, T = case["heads"], case["kv_heads"], case["head_dim"], case["page"], sum(news)
    if s["op"] == "append":
        # the definition rounds each product and each sum of the rotation to 32 bits, and the scale to 16
        x = s["qkv"].double().view(T, H + 2 * Hkv, hd // 2, 2)
        c, n = (s[w].double()[s["row_at"]][:, None] for w in ("cos", "sin"))
        r32 = lambda y: y.float().double()  # noqa: E731
        y = x.clone()
        y[:, : H + Hkv, :, 0] = r32(r32(x[:, : H + Hkv, :, 0] * c) - r32(x[:, : H + Hkv, :, 1] * n))
        y[:, : H + Hkv, :, 1] = r32(r32(x[:, : H + Hkv, :, 0] * n) + r32(x[:, : H + Hkv, :, 1] * c))
        y = y.view(T, H + 2 * Hkv, hd)
        z = y[:, H:].reshape(-1, GROUP)
        low, high = z.amin(1), z.amax(1)
        far = torch.where(-low == high, z.gather(1, z.abs().argmax(1, keepdim=True))[:, 0], torch.where(-low > high, low, high))
        d = torch.clamp((far / -8).half().double(), -65504, 65504)[:, None]
        code = torch.where(d == 0, 0.0, torch.clamp(torch.round(z / torch.where(d == 0, 1.0, d)), -8, 7))
        held = (code * d).view(T, 2 * Hkv, hd)
        q = x[:, :H, :, 0] * c - x[:, :H, :, 1] * n, x[:, :H, :, 0] * n + x[:, :H, :, 1] * c
        return dict(q=torch.stack(q, -1).reshape(T, H * hd), k=held[:, :Hkv].reshape(T, -1), v=held[:, Hkv:].reshape(T, -1))
    out, lse, at = [], [], 0
    for b, (n, length) in enumerate(zip(news, lens)):
        used = s["table"][b, : -(-length // page)].long()
        kv = []
        for name in ("k", "v"):
            raw = s[name + "_pool"][used]
            half = page * hd // 2
            byte = raw[:, :, :half].reshape(len(used), Hkv, page, hd // 2, 1)
            code = torch.cat((byte % 16, byte // 16), -1).double().reshape(len(used), Hkv, page, hd // GROUP, GROUP) - 8
            d = raw[:, :, half:].contiguous().view(torch.float16).double().view(len(used), Hkv, page, hd // GROUP, 1)
            kv.append((code * d).view(len(used), Hkv, page, hd).transpose(0, 1).reshape(Hkv, -1, hd)[:, :length])
        q = s["qkv"][at:at + n].double().view(n, Hkv, H // Hkv, hd)
        at += n
        x = torch.einsum("nhgd,hld->hgnl", q, kv[0]) / math.sqrt(hd)
        i = torch.arange(length, device=x.device)
        x = torch.where(i[None, :] <= (length - n + torch.arange(n, device=x.device))[:, None], x, float("-inf"))
        lse.append(torch.logsumexp(x, -1).permute(2, 0, 1).reshape(n, H))
        out.append(torch.einsum("hgnl,hld->nhgd", torch.softmax(x, -1), kv[1]).reshape(n, H * hd))
    return dict(out=torch.cat(out), lse=torch.cat(lse))
