"""The operators of the paged 4-bit K/V cache and of token scoring, as cases to time and to compare.

Three operators of brewference_b200.api:

  append    KvCache.append: head-wise RMSNorm (optional), position rotation of q and k, and k and v stored in the
            paged cache as blocks of 32 four-bit values with one fp16 scale (the Q4_0 rule)
  attend    KvCache.attend: softmax(q k^T) v over that cache, for single tokens and for prompt chunks, causal,
            with an optional sliding window and shared key/value heads
  logprobs  Logits.logprobs_device: log probabilities of given tokens, the entropy of each row and its top
            alternatives

`own` selects between their plain form (elementary torch operations) and the framework's calls.  Head layouts,
windows and vocabularies are those of brewference_b200/config.py.
"""
import math

import torch

if torch.cuda.is_available():
    torch.backends.cuda.matmul.allow_tf32 = False

own = False

EPS = 1e-6
HALF, INTERLEAVED = "half", "interleaved"


# ---- cases ------------------------------------------------------------------------------------------------------------

def _append(name, seqs, rows, pos, heads, kv_heads, head, rope, norm, page):
    return {"name": name, "op": "append", "seqs": seqs, "rows": rows, "pos": pos, "heads": heads, "kv_heads": kv_heads,
            "head": head, "rope": rope, "norm": norm, "page": page}


def _attend(name, seqs, rows, ctx, ragged, heads, kv_heads, head, window, page):
    return {"name": name, "op": "attend", "seqs": seqs, "rows": rows, "ctx": ctx, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head": head, "window": window, "page": page}


def _logprobs(name, rows, vocab, top, masked):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "masked": masked}


def listed():
    return [
        # one decode step of a small model: the call's latency
        _append("append one token", 1, 1, 700, 9, 3, 64, INTERLEAVED, False, 64),
        # one decode step of a served batch
        _append("append a batch", 32, 1, 3000, 28, 4, 128, HALF, False, 64),
        # prompts of many lengths entering the cache together, q and k normalised on the way
        _append("append prompts", 24, 601, 1500, 16, 8, 128, HALF, True, 32),
        # a short chat, one token: latency
        _attend("attend short", 1, 1, 333, False, 9, 3, 64, 0, 64),
        # one long document, one token: the work split over the positions
        _attend("attend long", 1, 1, 131071, False, 16, 8, 128, 0, 64),
        # a served batch of equal lengths, the largest read
        _attend("attend a batch", 128, 1, 8192, False, 28, 4, 128, 0, 64),
        # a served batch of unequal lengths, small pages
        _attend("attend a ragged batch", 32, 1, 32768, True, 28, 4, 128, 0, 16),
        # local layers: only the window's pages are read, heads of 256
        _attend("attend a window", 16, 1, 4001, True, 4, 1, 256, 512, 32),
        # the last chunk of a 4096-token prompt
        _attend("attend a prompt chunk", 1, 512, 4096, False, 16, 8, 128, 0, 64),
        # prompts of unequal lengths, parts of them in the cache already
        _attend("attend ragged prompts", 6, 700, 2000, True, 28, 4, 128, 0, 64),
        # the log probability of one sampled token with its alternatives: latency
        _logprobs("score one token", 1, 49152, 5, False),
        # a document scored row by row against the vocabulary
        _logprobs("score a document", 1777, 151936, 20, True),
    ]


_SHAPES = [(9, 3, 64), (16, 8, 128), (4, 1, 256), (28, 4, 128), (8, 4, 256), (16, 4, 128), (32, 32, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    if op == "logprobs":
        c = _logprobs("", _log(rng, 1, 1777), rng.choice([32000, 49152, 128256, 151936, 152064, 262144, _log(rng, 257, 262144)]),
                      rng.choice([0, 1, 5, 20, 32]), rng.random() < 0.5)
    else:
        heads, kv_heads, head = rng.choice(_SHAPES)
        page = rng.choice([16, 32, 64, 128])
        if op == "append":
            rows = 1 if rng.random() < 0.4 else _log(rng, 2, 1500)
            c = _append("", _log(rng, 1, 64), rows, _log(rng, 1, 100000), heads, kv_heads, head,
                        rng.choice([HALF, INTERLEAVED]), rng.random() < 0.5, page)
        else:
            rows = 1 if rng.random() < 0.6 else _log(rng, 2, 1024)
            c = _attend("", _log(rng, 1, 128), rows, rows + _log(rng, 1, 131072), rng.random() < 0.5, heads, kv_heads, head,
                        rng.choice([0, 0, 0, 512, 4096, _log(rng, 1, 2000)]), page)
    del c["name"]
    return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _padded(case):
    """Values that the plain form holds at once: a drawn case is one that it can run."""
    if case["op"] != "attend":
        return 0
    span = max(n - f for n, f in zip(_lens(case), _firsts(case)))
    return case["seqs"] * span * max(2 * case["kv_heads"] * case["head"], case["rows"] * case["heads"])


def draw(rng):
    top = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("append", "attend", "logprobs")}
    most = max(_padded(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= top[c["op"]] and _padded(c) <= most:
            return c


# Unequal sizes of a batch, from the case alone: the first is the largest.
def _share(i):
    return 1.0 if i == 0 else ((0.6180339887 * i) % 1.0) ** 2


def _rows(case):
    if case["rows"] == 1:
        return [1] * case["seqs"]
    if case["op"] == "attend" and not case["ragged"]:
        return [case["rows"]] * case["seqs"]
    return [max(1, int(case["rows"] * _share(i))) for i in range(case["seqs"])]


def _starts(case):
    """append: the position of each sequence's first new row."""
    return [int(case["pos"] * _share(case["seqs"] - i)) for i in range(case["seqs"])]


def _lens(case):
    """attend: keys of each sequence, its own query rows' among them."""
    if not case["ragged"]:
        return [case["ctx"]] * case["seqs"]
    return [max(r, int(case["ctx"] * _share(i))) for i, r in enumerate(_rows(case))]


def _firsts(case):
    """attend: the first key that any row of each sequence sees."""
    w = case["window"]
    return [max(0, n - r - w + 1) if w else 0 for n, r in zip(_lens(case), _rows(case))]


def work(case):
    if case["op"] == "logprobs":
        t, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * t * v + t * (4 + 8 + 8 * k), "flops": 6 * t * v}
    hd, hq, hk = case["head"], case["heads"], case["kv_heads"]
    rows = _rows(case)
    t = sum(rows)
    kv_row = 2 * hk * (hd // 2 + hd // 16)   # one position's k and v: 4 bits a value and fp16 scales
    if case["op"] == "append":
        # q, k and v read, q and the blocks written, the stored values handed back
        return {"bytes": t * (4 * hd * (2 * hq + 4 * hk) + 2 * kv_row), "flops": t * hd * (8 * hq + 20 * hk)}
    w, pairs, span = case["window"], 0, 0
    for r, n, f in zip(rows, _lens(case), _firsts(case)):
        span += n - f
        for j in range(r):
            p = n - r + j + 1
            pairs += min(p, w) if w else p
    return {"bytes": span * kv_row + 8 * t * hq * hd, "flops": 4 * pairs * hq * hd}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = dict(case)
    if case["op"] == "logprobs":
        t, v = case["rows"], case["vocab"]
        logits = torch.randn(t, v, generator=g, device="cuda") * 2.5
        if case["masked"]:   # tokens that a grammar forbids
            logits[torch.rand(t, v, generator=g, device="cuda") < 0.3] = -math.inf
        state["logits"] = logits
        state["tokens"] = torch.randint(0, v, (t,), generator=g, device="cuda", dtype=torch.int32)
        state["out"] = (torch.empty(t, device="cuda"), torch.empty(t, device="cuda"),
                        torch.empty(t, case["top"], dtype=torch.int32, device="cuda"),
                        torch.empty(t, case["top"], device="cuda"))
        return state
    hd, hq, hk, page, n = case["head"], case["heads"], case["kv_heads"], case["page"], case["seqs"]
    rows = _rows(case)
    t = sum(rows)
    starts = _starts(case) if case["op"] == "append" else [m - r for m, r in zip(_lens(case), rows)]
    lens = [s + r for s, r in zip(starts, rows)]
    most = max(lens)
    # the plain form's cache: pools of pages, and each sequence's pages in no order
    per_seq = [-(-m // page) for m in lens]
    ids = torch.randperm(sum(per_seq), generator=g, device="cuda", dtype=torch.int32)
    table = torch.zeros(n, -(-most // page), dtype=torch.int32, device="cuda")
    at = 0
    for i, m in enumerate(per_seq):
        table[i, :m] = ids[at:at + m]
        at += m
    slots = sum(per_seq) * page
    pool = {"kq": torch.zeros(slots, hk, hd // 2, dtype=torch.uint8, device="cuda"),
            "kd": torch.zeros(slots, hk, hd // 32, dtype=torch.float16, device="cuda"),
            "vq": torch.zeros(slots, hk, hd // 2, dtype=torch.uint8, device="cuda"),
            "vd": torch.zeros(slots, hk, hd // 32, dtype=torch.float16, device="cuda")}
    state.update(table=table, pool=pool, t=t, max_rows=max(rows), span=0)
    state["seq"] = torch.arange(n, dtype=torch.int32, device="cuda")
    state["pos"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    offs = [0]
    for r in rows:
        offs.append(offs[-1] + r)
    state["row_start"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
    # each query row's sequence and its place in it
    reps = torch.tensor(rows, device="cuda")
    state["row_seq"] = torch.repeat_interleave(torch.arange(n, device="cuda"), reps)
    state["row_in"] = torch.arange(t, device="cuda") - state["row_start"][:-1].long()[state["row_seq"]]
    state["q"] = torch.randn(t, hq, hd, generator=g, device="cuda") * 1.3
    if own:
        from brewference_b200 import api
        kv = api.KvCache(1, hq, hk, hd, n, most, page_tokens=page, n_pages=sum(per_seq))
        for part in (3, 2, 1):   # the sequences grow in turns, as served ones do
            for i, m in enumerate(lens):
                kv.reserve(i, -(-m // part))
        state["kv"] = kv
        state["rows_c"] = api.KvRows(state["seq"].data_ptr(), state["pos"].data_ptr(), n, t, max(rows),
                                     state["row_start"].data_ptr())
        state["workspace"] = torch.zeros(kv.workspace_bytes(), dtype=torch.uint8, device="cuda")
    if case["op"] == "append":
        state["k"] = torch.randn(t, hk, hd, generator=g, device="cuda") * 1.7
        state["v"] = torch.randn(t, hk, hd, generator=g, device="cuda")
        state["theta"] = 1e6 if case["rope"] == HALF else 1e5
        state["wq"] = state["wk"] = None
        if case["norm"]:
            state["wq"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda")
            state["wk"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda")
        state["out"] = (torch.empty(t, hq, hd, device="cuda"), torch.empty(t, hk, hd, device="cuda"),
                        torch.empty(t, hk, hd, device="cuda"))
        if own:
            state["rope_c"] = api.KvRope(api.ROPE_HALF if case["rope"] == HALF else api.ROPE_INTERLEAVED, state["theta"],
                                         1.0, state["wq"].data_ptr() if case["norm"] else 0,
                                         state["wk"].data_ptr() if case["norm"] else 0, EPS)
        return state
    state["first"] = torch.tensor(_firsts(case), device="cuda")
    state["lens"] = torch.tensor(lens, device="cuda")
    state["span"] = max(m - f for m, f in zip(lens, _firsts(case)))
    state["out"] = torch.empty(t, hq, hd, device="cuda")
    # what the cache holds: keys with a few strong channels, values of one size
    gain = torch.exp(0.5 * torch.randn(hk, hd, generator=g, device="cuda"))
    for i, m in enumerate(lens):
        for p0 in range(0, m, 32768):
            p1 = min(m, p0 + 32768)
            k = torch.randn(p1 - p0, hk, hd, generator=g, device="cuda") * gain
            v = torch.randn(p1 - p0, hk, hd, generator=g, device="cuda")
            p = torch.arange(p0, p1, device="cuda")
            slot = table[i][p // page].long() * page + p % page
            _store(pool, slot, k, v)
            if own:
                one = torch.tensor([i, p0], dtype=torch.int32, device="cuda")
                offs = torch.tensor([0, p1 - p0], dtype=torch.int32, device="cuda")
                kv.append(0, 0, 0, 0, k.data_ptr(), v.data_ptr(), hk * hd,
                          api.KvRows(one.data_ptr(), one.data_ptr() + 4, 1, p1 - p0, p1 - p0, offs.data_ptr()), None)
                torch.cuda.synchronize()
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _quantize(x):
    """Blocks of 32: d = -(the value of largest magnitude) / 8 and q = floor(x / d + 8.5) in 0..15, in 32 bits."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    m = torch.gather(b, -1, b.abs().argmax(-1, keepdim=True))
    d = (m / -8).clamp(-65504, 65504)
    inv = torch.where(d == 0, 0.0, 1.0 / d)
    q = torch.trunc(b * inv + 8.5).clamp(0, 15).to(torch.uint8).reshape(x.shape)
    return q, d.squeeze(-1).half()


def _store(pool, slot, k, v):
    for name, x in (("k", k), ("v", v)):
        q, d = _quantize(x)
        pool[name + "q"][slot] = q[..., 0::2] | (q[..., 1::2] << 4)
        pool[name + "d"][slot] = d


def _load(pool, name, slot):
    """The values that the blocks of these slots stand for, in 32 bits."""
    q = pool[name + "q"][slot]
    x = torch.stack((q & 15, q >> 4), -1).float() - 8
    d = pool[name + "d"][slot].float()
    return (x.reshape(*d.shape, 32) * d.unsqueeze(-1)).reshape(*q.shape[:-1], 2 * q.shape[-1])


def _rotated(s, x, w):
    """RMSNorm of each head and the rotation by its row's position, in 64 bits (a stored value may lie next to a border)."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    hd = x.shape[-1]
    i = torch.arange(hd // 2, device=x.device, dtype=torch.float64)
    pos = (s["pos"].long()[s["row_seq"]] + s["row_in"]).double()
    angle = pos[:, None] * torch.pow(torch.tensor(s["theta"], dtype=torch.float64, device=x.device), -2 * i / hd)
    c, n = angle.cos()[:, None], angle.sin()[:, None]
    if s["rope"] == HALF:
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat((a * c - b * n, a * n + b * c), -1).float()
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2).float()


def _append_plain(s):
    q, k = _rotated(s, s["q"], s["wq"]), _rotated(s, s["k"], s["wk"])
    p = s["pos"].long()[s["row_seq"]] + s["row_in"]
    slot = s["table"][s["row_seq"], p // s["page"]].long() * s["page"] + p % s["page"]
    _store(s["pool"], slot, k, s["v"])
    return q, _load(s["pool"], "k", slot), _load(s["pool"], "v", slot)


def _attend_plain(s):
    n, hd, hk, r = s["seqs"], s["head"], s["kv_heads"], s["max_rows"]
    group = s["heads"] // hk
    # keys and values of every sequence, padded to the longest
    kpos = s["first"][:, None] + torch.arange(s["span"], device="cuda")
    there = kpos < s["lens"][:, None]
    p = torch.where(there, kpos, 0)
    slot = torch.gather(s["table"], 1, p // s["page"]).long() * s["page"] + p % s["page"]
    k, v = _load(s["pool"], "k", slot).transpose(1, 2), _load(s["pool"], "v", slot).transpose(1, 2)
    # query rows, padded likewise: [sequence, kv head, row * group, head size]
    ri = (s["row_start"][:-1].long()[:, None] + torch.arange(r, device="cuda")).clamp(max=s["t"] - 1)
    q = s["q"][ri].reshape(n, r, hk, group, hd).permute(0, 2, 1, 3, 4).reshape(n, hk, r * group, hd)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    qpos = (s["pos"].long()[:, None] + torch.arange(r, device="cuda")).repeat_interleave(group, 1)[:, :, None]
    seen = there[:, None] & (kpos[:, None] <= qpos)
    if s["window"]:
        seen &= kpos[:, None] > qpos - s["window"]
    x = torch.where(seen[:, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0, m))   # a padding row may see no key
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.reshape(n, hk, r, group, hd).permute(0, 2, 1, 3, 4).reshape(n, r, hk * group, hd)
    return o[s["row_seq"], s["row_in"]]


def _logprobs_plain(s):
    x = s["logits"]
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    z = e.sum(-1, keepdim=True)
    lse = torch.log(z)
    entropy = lse[:, 0] - torch.where(e > 0, e * y, 0.0).sum(-1) / z[:, 0]
    logprob = (torch.gather(y, 1, s["tokens"].long()[:, None]) - lse)[:, 0]
    # whole numbers in the order of (logit, lowest index first), so that no two are equal
    bits = y.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32 + torch.arange(x.shape[1] - 1, -1, -1, device="cuda")
    order = torch.topk(key, s["top"], -1)[1]
    return logprob, entropy, order.int(), torch.gather(y, 1, order) - lse


def run(state):
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "logprobs": _logprobs_plain}[state["op"]](state)
    from brewference_b200 import api
    stream = torch.cuda.current_stream().cuda_stream
    out = state["out"]
    if state["op"] == "logprobs":
        t, v = state["logits"].shape
        api.Logits.logprobs_device(state["logits"].data_ptr(), v, v, t, state["tokens"].data_ptr(), out[0].data_ptr(),
                                   out[1].data_ptr(), state["top"], out[2].data_ptr(), out[3].data_ptr(), stream)
        return out
    kv, hd = state["kv"], state["head"]
    qw, kw = state["heads"] * hd, state["kv_heads"] * hd
    if state["op"] == "append":
        kv.append(0, out[0].data_ptr(), state["q"].data_ptr(), qw, state["k"].data_ptr(), state["v"].data_ptr(), kw,
                  state["rows_c"], state["rope_c"], stream)
        kv.read(0, out[1].data_ptr(), out[2].data_ptr(), kw, state["rows_c"], stream)
        return out
    kv.attend(0, out.data_ptr(), qw, state["q"].data_ptr(), qw, state["rows_c"], state["window"],
              state["workspace"].data_ptr(), stream=stream)
    return out


# ---- the definitions, in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        lp, ent, ids, tops = [], [], [], []
        for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            x = x.double()
            logp = x - torch.logsumexp(x, -1, keepdim=True)
            lp.append(torch.gather(logp, 1, t.long()[:, None])[:, 0])
            ent.append(-torch.special.xlogy(logp.exp(), logp.exp()).sum(-1))
            tops.append(torch.topk(logp, case["top"], -1)[0])
        return torch.cat(lp), torch.cat(ent), None, torch.cat(tops)
    hd, hq, hk = case["head"], case["heads"], case["kv_heads"]
    if case["op"] == "append":
        pos = torch.cat([p + torch.arange(r, device="cuda") for p, r in zip(_starts(case), _rows(case))]).double()
        freq = torch.exp(torch.arange(0, hd, 2, device="cuda").double() * (-math.log(s["theta"]) / hd))
        turn = torch.polar(torch.ones_like(freq).expand(len(pos), -1), pos[:, None] * freq)[:, None]

        def turned(x, w):
            x = x.double()
            if w is not None:
                x = x * (x.square().sum(-1, keepdim=True) / hd + EPS).rsqrt() * w.double()
            if case["rope"] == HALF:
                z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
                return torch.cat((z.real, z.imag), -1)
            return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)

        def held(x):
            """What the cache holds of x, which reaches it in 32 bits."""
            b = x.float().unflatten(-1, (-1, 32))
            hi, lo = b.max(-1, keepdim=True), b.min(-1, keepdim=True)
            up = (hi[0] > -lo[0]) | ((hi[0] == -lo[0]) & (b.abs().max(-1, keepdim=True)[1] == hi[1]))
            d = torch.where(up, hi[0], lo[0]) * -0.125
            code = torch.floor(torch.where(d != 0, b * d.reciprocal(), 0) + 8.5).clamp(max=15)
            return ((code - 8).double() * d.half().double()).flatten(-2)

        return turned(s["q"], s["wq"]), held(turned(s["k"], s["wk"])), held(s["v"])
    pool, outs, at = s["pool"], [], 0
    group, w = hq // hk, case["window"]
    for i, (r, m, f) in enumerate(zip(_rows(case), _lens(case), _firsts(case))):
        p = torch.arange(f, m, device="cuda")
        slot = s["table"][i][p // case["page"]].long() * case["page"] + p % case["page"]

        def values(name):
            q = pool[name + "q"][slot]
            x = torch.empty(len(p), hk, hd, dtype=torch.float64, device="cuda")
            x[..., 0::2], x[..., 1::2] = (q % 16).double() - 8, (q // 16).double() - 8
            return x * pool[name + "d"][slot].double().repeat_interleave(32, -1)

        k, v = values("k"), values("v")
        qi = s["q"][at:at + r].double().view(r, hk, group, hd)
        at += r
        x = torch.einsum("rhgd,khd->hgrk", qi, k) / math.sqrt(hd)
        last = m - r + torch.arange(r, device="cuda")[:, None]
        hidden = p > last
        if w:
            hidden = hidden | (p <= last - w)
        o = torch.einsum("hgrk,khd->rhgd", torch.softmax(x.masked_fill(hidden, -math.inf), -1), v)
        outs.append(o.reshape(r, hq, hd))
    return torch.cat(outs)
