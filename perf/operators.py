"""Operators around a KV pool held in 8 bits, and attention with a sliding window and sinks, as cases that can be timed.

A program that serves long contexts keeps the K/V rows of all requests in one pool, a slot per token.  Five kinds of calls:
"write" puts the rows of new tokens into a pool of e4m3 values with a power-of-two scale for each token and head, "read"
brings the rows of a context back as 16-bit K/V for the next chunk of a prompt, "decode8" attends from one new token per
request to such a pool, "decode" does so over a pool in 16 bits where every token sees a window of the last tokens and a few
first ones (sinks), "prefill" is that window over the tokens of prompts.

listed() holds ordinary points of these kinds, draw() gives others of the same ranges.  Lengths come from the case alone,
values and slot numbers from the seed.  Where `own` is false, run() computes the plain forms in float32.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
PAD = 2147483647  # unused entries of the request table


def listed():
    return [
        # the new tokens of a decode step of eight requests are written: the smallest write, where the launch counts
        dict(name="write_8_tokens", kind="write", tokens=8, kv_heads=8, head_dim=128, dtype="f16"),
        # the rows of a long prompt, MHA with 32 heads in bfloat16, odd length
        dict(name="write_16383_mha", kind="write", tokens=16383, kv_heads=32, head_dim=128, dtype="bf16"),
        # contexts of a few ragged requests are read back in front of their next chunk
        dict(name="read_5_ragged", kind="read", batch=5, shortest=1, longest=1500, kv_heads=8, head_dim=128, dtype="f16", lens=1),
        # one request's long context is read back
        dict(name="read_131072", kind="read", batch=1, shortest=131072, longest=131072, kv_heads=8, head_dim=128, dtype="bf16", lens=2),
        # one user's decode step over the 8-bit pool: a single request, where latency counts
        dict(name="decode8_1x2047", kind="decode8", batch=1, shortest=2047, longest=2047, q_heads=32, kv_heads=8, head_dim=128, dtype="f16",
             window=0, sinks=0, lens=3),
        # the decode step of a full batch of long requests over the 8-bit pool
        dict(name="decode8_64_long", kind="decode8", batch=64, shortest=4096, longest=32768, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", window=0, sinks=0, lens=4),
        # two requests of very long contexts, MHA in bfloat16, a window of some thousand tokens: the latency of a long model in chat
        dict(name="decode8_2_window_mha", kind="decode8", batch=2, shortest=60000, longest=131072, q_heads=32, kv_heads=32,
             head_dim=128, dtype="bf16", window=4096, sinks=4, lens=5),
        # a window over the 16-bit pool for one request that is a little longer than the window
        dict(name="decode_1_window", kind="decode", batch=1, shortest=1100, longest=1100, q_heads=32, kv_heads=8, head_dim=128, dtype="f16",
             window=1024, sinks=4, lens=6),
        # a large batch of requests behind one window, some shorter than it
        dict(name="decode_96_window", kind="decode", batch=96, shortest=700, longest=16384, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16",
             window=4096, sinks=64, lens=7),
        # a short prompt with a small window: the smallest prefill call
        dict(name="prefill_1x777", kind="prefill", batch=1, shortest=777, longest=777, context=0, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", window=256, sinks=4, lens=8),
        # a batch of ragged prompts, MHA in bfloat16
        dict(name="prefill_6_ragged_mha", kind="prefill", batch=6, shortest=300, longest=4000, context=0, q_heads=32, kv_heads=32, head_dim=128,
             dtype="bf16", window=1000, sinks=0, lens=9),
        # one long prompt behind a window of some thousand tokens
        dict(name="prefill_1x32768", kind="prefill", batch=1, shortest=32768, longest=32768, context=0, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", window=4096, sinks=16, lens=10),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode8", "decode", "prefill"])
    heads = [(32, 8), (32, 32), (8, 1), (16, 2), (28, 4)]
    while True:
        hq, hkv = rng.choice(heads)
        c = dict(kind=kind, kv_heads=hkv, head_dim=rng.choice([128, 128, 128, 64]), dtype=rng.choice(["f16", "bf16"]))
        if kind == "write":
            c.update(tokens=_log_int(rng, 1, 16383))
        else:
            batch = _log_int(rng, 1, 6 if kind == "prefill" else 96)
            longest = _log_int(rng, 64, 131072)
            c.update(batch=batch, longest=longest, shortest=rng.randint(1, longest), lens=rng.randint(100, 10 ** 6))
        if kind in ("decode8", "decode", "prefill"):
            c.update(q_heads=hq, window=_log_int(rng, 32, 8192), sinks=rng.choice([0, 1, 4, rng.randint(2, 128)]))
        if kind == "decode8" and rng.random() < 0.5:
            c.update(window=0, sinks=0)
        if kind == "prefill":
            c.update(context=rng.choice([0, 0, rng.randint(1, 4000)]))
        w, most = work(c), max((work(d) for d in listed() if d["kind"] == kind), key=lambda w: w["flops"] + w["bytes"])
        room = sum(_lens(c)) * 2 * hkv * c["head_dim"] if kind in ("read", "decode8", "decode") else 0  # elements of the pool
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and room <= 3e9 and _plain_scores(c) <= 6e9:
            return c


def _plain_scores(c):
    """Scores that the plain form holds at once."""
    if c["kind"] == "prefill":
        n = c["longest"] + _block(c["window"])
        return c["batch"] * c["q_heads"] * n * (c["window"] + _block(c["window"]) + c["sinks"])
    if c["kind"] in ("decode8", "decode"):
        return c["batch"] * (c["q_heads"] + 2 * c["kv_heads"] * c["head_dim"]) * _columns(c, c["longest"])
    return 0


def _lens(c):
    """The batch's lengths, the longest and the shortest among them."""
    r = random.Random(c["lens"])
    lens = [r.randint(c["shortest"], c["longest"]) for _ in range(c["batch"])]
    lens[-1] = c["shortest"]
    lens[0] = c["longest"]
    return lens


def _columns(c, longest):
    return min(longest, c["window"] + c["sinks"]) if c["window"] else longest


def _pairs(c):
    """Pairs of a query and a key that it sees."""
    n = 0
    w, s = c["window"], c["sinks"]
    for t in _lens(c):
        if c["kind"] == "prefill":
            p0, p1 = c["context"], c["context"] + t  # positions of the queries
            full = lambda p: p * (p + 1) // 2  # noqa: E731  (pairs of the first p positions under a causal mask alone)
            seen = lambda p: full(min(p, w)) + max(0, p - w) * w  # noqa: E731
            kept = lambda p: full(min(max(0, p - w), s)) + max(0, p - w - s) * s  # noqa: E731
            n += seen(p1) - seen(p0) + kept(p1) - kept(p0)
        else:
            n += min(t, w + s) if w else t
    return n


def work(case):
    c = case
    row = 2 * c["kv_heads"]
    d = c["head_dim"]
    if c["kind"] == "write":
        return {"bytes": c["tokens"] * (row * (3 * d + 1) + 8), "flops": 0}
    if c["kind"] == "read":
        return {"bytes": sum(_lens(c)) * (row * (3 * d + 1) + 4), "flops": 0}
    n = _pairs(c)
    if c["kind"] == "prefill":
        t = sum(_lens(c))
        return {"bytes": t * (c["q_heads"] * (4 * d + 4)) + (t + c["batch"] * c["context"]) * row * 2 * d, "flops": 4 * d * c["q_heads"] * n}
    per_row = d + 1 if c["kind"] == "decode8" else 2 * d
    return {"bytes": n * (row * per_row + 4) + c["batch"] * c["q_heads"] * (6 * d + 4), "flops": 4 * d * c["q_heads"] * n}


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, tokens, kv_heads, head_dim, dtype):
    """K heads then V heads of `tokens` tokens: K with a few strong channels, V of a size that differs from token to token."""
    x = torch.randn(tokens, 2 * kv_heads, head_dim, generator=g, device=DEV, dtype=torch.float32)
    channel = torch.rand(kv_heads, head_dim, generator=g, device=DEV)
    x[:, :kv_heads] *= 0.5 + 2.5 * (channel > 0.95)
    x[:, kv_heads:] *= torch.exp(0.5 * torch.randn(tokens, 1, 1, generator=g, device=DEV))
    return x.to(dtype)


def _quantised(x):
    """(e4m3 values, exponents + 127) of rows [.., head_dim], by a power-of-two scale for each row.  Every step but the last is exact in
    float32: frexp, the product with a power of two; NaN stands for what is not finite."""
    x = x.float()
    amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)  # 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    q = (x * torch.ldexp(torch.ones_like(amax), -e)[..., None]).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8)


def _pool8(g, slots, c):
    """A pool in 8 bits of rows as they come, some at a time."""
    h, d = 2 * c["kv_heads"], c["head_dim"]
    pool = torch.empty(slots, h, d, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.empty(slots, h, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 28) // (h * d))
    for i in range(0, slots, step):
        n = min(step, slots - i)
        q, s = _quantised(_rows(g, n, c["kv_heads"], d, DTYPES[c["dtype"]]))
        pool.view(torch.uint8)[i:i + n] = q.view(torch.uint8)
        scales[i:i + n] = s
    return pool, scales


def _pool16(g, slots, c):
    pool = torch.empty(slots, 2 * c["kv_heads"], c["head_dim"], dtype=DTYPES[c["dtype"]], device=DEV)
    step = max(1, (1 << 28) // (2 * c["kv_heads"] * c["head_dim"]))
    for i in range(0, slots, step):
        n = min(step, slots - i)
        pool[i:i + n] = _rows(g, n, c["kv_heads"], c["head_dim"], DTYPES[c["dtype"]])
    return pool


def _table(g, lens, slots):
    """Scattered slots of the requests' tokens, the requests in no order of the table's rows; unused entries as the request table has them."""
    batch = len(lens)
    table = torch.full((batch + 3, max(lens) + 5), PAD, dtype=torch.int32, device=DEV)
    req = torch.randperm(batch + 3, generator=g, device=DEV)[:batch].to(torch.int32)
    slot = torch.randperm(slots, generator=g, device=DEV).to(torch.int32)
    at = 0
    for b, n in enumerate(lens):
        table[int(req[b]), :n] = slot[at:at + n]
        at += n
    return table, req


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lens):
    return _ints([sum(lens[:b]) for b in range(len(lens))])


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)
    s = dict(case=c)
    h, d, dtype = 2 * c["kv_heads"], c["head_dim"], DTYPES[c["dtype"]]
    if c["kind"] == "write":
        t = c["tokens"]
        slots = t + t // 4 + 16
        s.update(src=_rows(g, t, c["kv_heads"], d, dtype), index=torch.randperm(slots, generator=g, device=DEV)[:t].contiguous(),
                 pool=torch.zeros(slots, h, d, device=DEV).to(torch.float8_e4m3fn), scales=torch.full((slots, h), 127, dtype=torch.uint8, device=DEV))
        return s
    lens = _lens(c)
    if c["kind"] == "prefill":
        keys = [n + c["context"] for n in lens]
        rows = _rows(g, sum(keys), c["kv_heads"], d, dtype)
        q = torch.randn(sum(lens), c["q_heads"], d, generator=g, device=DEV).to(dtype)
        s.update(q=q, k=rows[:, :c["kv_heads"]], v=rows[:, c["kv_heads"]:], o=torch.zeros_like(q),
                 lse=torch.zeros(sum(lens), c["q_heads"], device=DEV), q_start=_starts(lens), q_len=_ints(lens), q_first=_ints([c["context"]] * len(lens)),
                 kv_start=_starts(keys), kv_len=_ints(keys), kv_first=_ints([0] * len(lens)), longest=max(lens), shape=(lens, keys))
        return s
    slots = sum(lens) + sum(lens) // 8 + 32
    table, req = _table(g, lens, slots)
    s.update(table=table, req=req, len=_ints(lens), longest=max(lens))
    if c["kind"] in ("read", "decode8"):
        s["pool"], s["scales"] = _pool8(g, slots, c)
    else:
        s["pool"] = _pool16(g, slots, c)
    if c["kind"] == "read":
        s.update(start=_starts(lens), out=torch.zeros(sum(lens), h, d, dtype=dtype, device=DEV))
    else:
        s["q"] = torch.randn(c["batch"], c["q_heads"], d, generator=g, device=DEV).to(dtype)
    return s


# ------------------------------------------------------------------------------------------------ plain forms, float32
def _scale(scales):
    return (scales.int() << 23).view(torch.float32)[..., None]  # 2^(byte - 127), byte >= 1


def _values(pool, scales, slots):
    return pool.view(torch.uint8)[slots].view(torch.float8_e4m3fn).float() * _scale(scales[slots])


def _flat_slots(table, req, lens, longest):
    """Slots of the requests' tokens one request after the other."""
    pos = torch.arange(longest, device=DEV)
    return table[req.long(), :longest][pos[None] < lens[:, None]].long()


def _visible(c, lens, longest):
    """Positions that the last token of every request sees [batch, columns], and whether each exists; first the sinks, then the window."""
    i = torch.arange(_columns(c, longest), device=DEV)[None]
    n = lens.long()[:, None]
    if not c["window"]:
        return i.expand(n.shape[0], -1), i < n
    start = (n - c["window"]).clamp(min=c["sinks"])
    pos = torch.where(i < c["sinks"], i, start + i - c["sinks"])
    return pos, pos < n


def _softmax_sum(s, v):
    """(sum of v under the softmax of s, log of the sum of exponentials), over the last dimension of s."""
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    return p.matmul(v) / l, (m + torch.log(l)).squeeze(-1)


def _decode(c, s):
    pos, there = _visible(c, s["len"], s["longest"])
    slots = torch.where(there, s["table"][s["req"].long()].gather(1, pos.clamp(max=s["longest"] - 1)), torch.zeros_like(pos, dtype=torch.int32)).long()
    if c["kind"] == "decode8":
        rows = _values(s["pool"], s["scales"], slots)
    else:
        rows = s["pool"][slots].float()
    hkv, d = c["kv_heads"], c["head_dim"]
    q = s["q"].float().view(c["batch"], hkv, c["q_heads"] // hkv, d)
    k, v = rows[:, :, :hkv].permute(0, 2, 3, 1).contiguous(), rows[:, :, hkv:].permute(0, 2, 1, 3).contiguous()
    del rows
    x = q.matmul(k) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~there[:, None, None], -math.inf)
    o, lse = _softmax_sum(x, v)
    return o.reshape(c["batch"], c["q_heads"], d), lse.reshape(c["batch"], c["q_heads"])


def _block(window):
    return max(64, min(1024, window // 4 * 4))


def _windows(x, front, first, size, step, count):
    """[batch, count, heads, size, head_dim]: `size` rows from `first` - `front` on, `step` further from one to the next."""
    b, t, h, d = x.shape
    tail = max(0, first + (count - 1) * step + size - front - t)
    x = torch.cat([x.new_zeros(b, front, h, d), x, x.new_zeros(b, tail, h, d)], 1)[:, first:]
    return x.unfold(1, size, step)[:, :count].permute(0, 1, 2, 4, 3).contiguous()


def _prefill(c, s):
    """Queries in blocks, each against the rows that the windows of its first and last query span, and against the sinks."""
    lens, keys = s["shape"]
    hkv, hq, d, w, sinks, ctx = c["kv_heads"], c["q_heads"], c["head_dim"], c["window"], c["sinks"], c["context"]
    longest, step = max(lens), _block(c["window"])
    count = -(-longest // step)
    at = torch.arange(longest + ctx, device=DEV)[None]
    kept = at < s["kv_len"][:, None]
    row = (s["kv_start"][:, None] + torch.where(kept, at, 0)).long()
    k, v = s["k"][row].float(), s["v"][row].float()
    qi = torch.arange(count * step, device=DEV)[None]
    q_there = qi < s["q_len"][:, None]
    q_row = (s["q_start"][:, None] + torch.where(q_there, qi, 0)).long()
    q = s["q"][q_row].float().view(len(lens), count, step, hkv, hq // hkv, d).permute(0, 1, 3, 4, 2, 5).reshape(len(lens), count, hkv, -1, d)
    scale = 1.0 / math.sqrt(d)
    size = step + w - 1
    near = q.matmul(_windows(k, w - 1, ctx, size, step, count).transpose(-1, -2).contiguous()).view(len(lens), count, hkv, hq // hkv, step, size) * scale
    i, j = torch.arange(step, device=DEV)[:, None], torch.arange(size, device=DEV)[None]
    key = torch.arange(count, device=DEV)[:, None, None] * step + ctx - (w - 1) + j  # position of column j of a block
    seen = (j >= i) & (j <= i + w - 1) & (key >= 0)
    near = near.masked_fill(~seen[None, :, None, None], -math.inf)
    parts = [near]
    del near
    if sinks:
        first = min(sinks, longest + ctx)
        kk, vv = k[:, None, :first].permute(0, 1, 3, 2, 4).contiguous(), v[:, None, :first].permute(0, 1, 3, 2, 4).contiguous()
        far = q.matmul(kk.transpose(-1, -2).contiguous()).view(len(lens), count, hkv, hq // hkv, step, first) * scale
        q_pos = (ctx + torch.arange(count * step, device=DEV)).view(count, step, 1)
        far = far.masked_fill(~(torch.arange(first, device=DEV) <= q_pos - w)[None, :, None, None], -math.inf)
        parts.append(far)
        del far
    x = torch.cat(parts, -1) if sinks else parts[0]
    del parts
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - m)
    l = x.sum(-1, keepdim=True)
    flat = x.view(len(lens), count, hkv, -1, x.shape[-1])
    o = flat[..., :size].matmul(_windows(v, w - 1, ctx, size, step, count))
    if sinks:
        o = o + flat[..., size:].matmul(vv)
    o = o.view(len(lens), count, hkv, hq // hkv, step, d) / l
    lse = m + torch.log(l)
    turn = lambda t: t.permute(0, 1, 4, 2, 3, 5).reshape(len(lens), count * step, hq, -1)[q_there]  # noqa: E731
    return turn(o).to(s["q"].dtype), turn(lse).squeeze(-1)


def run(state):
    s, c = state, state["case"]
    if own:
        import loongserve_amd as lsa
        hkv = c["kv_heads"]
        if c["kind"] == "write":
            lsa.kv_scatter_fp8(s["src"], s["index"], s["pool"], s["scales"])
            return s["pool"], s["scales"]
        if c["kind"] == "read":
            lsa.kv_gather_fp8(s["pool"], s["scales"], s["table"], s["req"], s["len"], s["start"], s["longest"], s["out"])
            return s["out"]
        if c["kind"] == "decode8":
            return lsa.longserve_fp8_decode_attention(s["q"], s["table"], s["req"], s["len"], s["longest"], s["pool"][:, :hkv], s["pool"][:, hkv:],
                                                      s["scales"][:, :hkv], s["scales"][:, hkv:], window=c["window"] or None, sinks=c["sinks"])
        if c["kind"] == "decode":
            return lsa.longserve_window_decode_attention(s["q"], s["table"], s["req"], s["len"], s["longest"], s["pool"][:, :hkv], s["pool"][:, hkv:],
                                                         c["window"], sinks=c["sinks"])
        lsa.window_attention_fwd(s["q"], s["k"], s["v"], s["o"], s["q_start"], s["q_len"], s["q_first"], s["kv_start"], s["kv_len"], s["kv_first"],
                                 1, s["longest"], c["window"], sinks=c["sinks"], lse=s["lse"])
        return s["o"], s["lse"]
    if c["kind"] == "write":
        q, e = _quantised(s["src"])
        s["pool"].view(torch.uint8)[s["index"]] = q.view(torch.uint8)
        s["scales"][s["index"]] = e
        return s["pool"], s["scales"]
    if c["kind"] == "read":
        s["out"][:] = _values(s["pool"], s["scales"], _flat_slots(s["table"], s["req"], s["len"], s["longest"])).to(s["out"].dtype)
        return s["out"]
    if c["kind"] == "prefill":
        return _prefill(c, s)
    return _decode(c, s)


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _e4m3(x):
    """The e4m3 value nearest to each of x (|x| <= 448), ties to the even one: multiples of 2^(exponent - 3), of 2^-9 at the least."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return torch.round(x / step) * step


def exact(case, seed):
    """The definitions in float64, request by request and KV head by KV head."""
    c = case
    s = prepare(case, seed)
    hkv, d = c["kv_heads"], c["head_dim"]
    if c["kind"] == "write":
        pool, scales = s["pool"].double(), s["scales"].double()
        x = s["src"].double()
        e = torch.ceil(torch.log2(x.abs().amax(-1) / 448))
        e = torch.where(x.abs().amax(-1) > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(x.abs().amax(-1) <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        pool[s["index"]] = _e4m3(x / torch.exp2(e)[..., None])
        scales[s["index"]] = e + 127
        return pool, scales.long()
    lens = s["len"].tolist() if "len" in s else s["shape"][0]
    if c["kind"] in ("read", "decode8"):
        def rows_of(slots, heads):
            return s["pool"].view(torch.uint8)[slots, heads].view(torch.float8_e4m3fn).double() * torch.exp2(s["scales"][slots, heads].double() - 127)[..., None]
    if c["kind"] == "read":
        out = torch.empty(s["out"].shape, dtype=torch.float64, device=DEV)
        at = 0
        for b, n in enumerate(lens):
            slots = s["table"][int(s["req"][b]), :n].long()
            for h in range(2 * hkv):
                out[at:at + n, h] = rows_of(slots, h)
            at += n
        return out
    group = c["q_heads"] // hkv
    o = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=DEV)

    def attend(q, k, v, seen):
        x = (q @ k.T) / math.sqrt(d)
        x = x.masked_fill(~seen, -math.inf)
        l = torch.logsumexp(x, -1)
        return torch.exp(x - l[:, None]) @ v, l

    if c["kind"] != "prefill":
        for b, n in enumerate(lens):
            pos = torch.arange(n, device=DEV)
            if c["window"]:
                pos = pos[(pos >= n - c["window"]) | (pos < c["sinks"])]
            slots = s["table"][int(s["req"][b]), :n].long()[pos]
            for h in range(hkv):
                if c["kind"] == "decode8":
                    k, v = rows_of(slots, h), rows_of(slots, hkv + h)
                else:
                    k, v = s["pool"][slots, h].double(), s["pool"][slots, hkv + h].double()
                heads = slice(h * group, (h + 1) * group)
                o[b, heads], lse[b, heads] = attend(s["q"][b, heads].double(), k, v, torch.ones(1, len(pos), dtype=torch.bool, device=DEV))
        return o, lse
    if work(c)["flops"] > 4e12:
        return None
    q0 = k0 = 0
    w, sinks, ctx = c["window"], c["sinks"], c["context"]
    for n, m in zip(*s["shape"]):
        for i in range(0, n, 2048):
            r = min(2048, n - i)
            p = ctx + i + torch.arange(r, device=DEV)[:, None]
            low = max(0, ctx + i - w + 1)
            j = torch.arange(min(low, sinks), device=DEV)
            j = torch.cat([j, torch.arange(low, min(m, ctx + i + r), device=DEV)])[None]
            seen = (j <= p) & ((j > p - w) | (j < sinks))
            for h in range(hkv):
                k, v = s["k"][k0 + j[0], h].double(), s["v"][k0 + j[0], h].double()
                q = s["q"][q0 + i:q0 + i + r, h * group:(h + 1) * group].double()
                got, l = attend(q.reshape(-1, d), k, v, seen.repeat_interleave(group, 0))
                o[q0 + i:q0 + i + r, h * group:(h + 1) * group] = got.view(r, group, d)
                lse[q0 + i:q0 + i + r, h * group:(h + 1) * group] = l.view(r, group)
        q0 += n
        k0 += m
    return o, lse
